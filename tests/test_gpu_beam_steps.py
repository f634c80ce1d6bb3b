"""stg_beam_start / _advance / _reorder / _backtrace against plain loops: everything here is exact."""
import numpy as np
import pytest

from tests import beam_oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=512, max_vocab=4096, max_history=40, max_top_k=8)
    yield b
    b.close()


# ---- advance -------------------------------------------------------------------------------------------

def _candidates(rng, B, K, n, t, eos, odd):
    tok = rng.integers(3, 50, (B, n)).astype(np.int32)
    tok[rng.random((B, n)) < 0.3] = eos[0] if eos else 5
    if len(eos) > 1:
        tok[rng.random((B, n)) < 0.1] = eos[1]
    par = rng.integers(0, K, (B, n)).astype(np.int32)
    sc = -(1.2 * t + np.cumsum(rng.random((B, n)), 1)).astype(np.float32)
    if odd:
        tok[rng.random((B, n)) < 0.1] = -1
        par[rng.random((B, n)) < 0.1] = rng.choice([-1, K, 1 << 30])
        sc[rng.random((B, n)) < 0.1] = rng.choice([-np.inf, np.nan])
        sc[:, n // 2:] = np.round(sc[:, n // 2:])  # ties
    return tok, par, sc


def _same(search, rows, T):
    got = {k: getattr(search, k).cpu().numpy() for k in ("tokens", "parents", "scores", "steps", "done", "pool_scores", "pool_steps", "pool_parents",
                                                         "pool_tokens", "trail_tokens", "trail_parents")}
    for b, r in enumerate(rows):
        assert got["steps"][b] == r.steps and (got["done"][b] != 0) == r.done
        assert [(t, p) for t, p, _ in r.beams] == list(zip(got["tokens"][b].tolist(), got["parents"][b].tolist()))
        assert np.array_equal(got["scores"][b], np.array([s for _, _, s in r.beams], np.float32))
        pool = r.pool + [(np.float32(-np.inf), -1, -1, -1)] * (r.K - len(r.pool))
        assert np.array_equal(got["pool_scores"][b], np.array([p[0] for p in pool], np.float32))
        assert list(zip(got["pool_steps"][b].tolist(), got["pool_parents"][b].tolist(), got["pool_tokens"][b].tolist())) == [tuple(p[1:]) for p in pool]
        for t, row in enumerate(r.trail):
            assert list(zip(got["trail_tokens"][t, b].tolist(), got["trail_parents"][t, b].tolist())) == row


@pytest.mark.parametrize("B,K,n,T", [(1, 1, 1, 1), (1, 1, 2, 3), (3, 4, 8, 6), (5, 3, 7, 9), (64, 8, 16, 5), (7, 32, 128, 4), (16, 32, 32, 3), (2, 5, 128, 8)])
@pytest.mark.parametrize("penalty,early,odd", [(1.0, False, False), (0.0, True, False), (0.7, False, True), (2.0, False, False)])
def test_advance(bs, B, K, n, T, penalty, early, odd):
    import torch
    from opentail.stingray_b200 import BeamSearch

    rng = np.random.default_rng(B * 1000 + K * 10 + n)
    eos = [2, 1]
    search = BeamSearch(B, K, T, eos=eos, pad=9, length_penalty=penalty, early_stopping=early)
    norms = search.norms.cpu().tolist()
    for request in range(2):  # a second one in the same arrays
        bs.beam_start(search)
        rows = [beam_oracle.Search(K, T, eos, 9, norms, early) for _ in range(B)]
        _same(search, rows, T)
        for t in range(T + 1):  # once more than there is room for
            tok, par, sc = _candidates(rng, B, K, n, t, eos, odd)
            finish = t == T - 2 and request == 1
            bs.beam_advance(search, {"tokens": torch.from_numpy(tok).cuda(), "parents": torch.from_numpy(par).cuda(), "scores": torch.from_numpy(sc).cuda()},
                            finish=finish)
            for b, r in enumerate(rows):
                r.advance([(int(tok[b, i]), int(par[b, i]), sc[b, i]) for i in range(n)], finish)
            _same(search, rows, T)


def test_no_end_tokens_and_early_ends(bs):
    import torch
    from opentail.stingray_b200 import BeamSearch

    search = BeamSearch(2, 2, 4)
    bs.beam_start(search)
    c = {"tokens": torch.tensor([[2, 3, 4], [-1, -1, -1]], dtype=torch.int32, device="cuda"), "parents": torch.zeros((2, 3), dtype=torch.int32, device="cuda"),
         "scores": torch.tensor([[-1.0, -2.0, -3.0], [0, 0, 0]], device="cuda")}
    bs.beam_advance(search, c)
    assert search.tokens.tolist() == [[2, 3], [0, 0]] and search.done.tolist() == [0, 1]  # nothing goes on in the second
    assert search.pool_steps.tolist() == [[-1, -1], [-1, -1]] and search.steps.tolist() == [1, 1]
    # every candidate ends
    search = BeamSearch(1, 3, 4, eos=[7])
    bs.beam_start(search)
    bs.beam_advance(search, {"tokens": torch.full((1, 6), 7, dtype=torch.int32, device="cuda"), "parents": torch.zeros((1, 6), dtype=torch.int32, device="cuda"),
                             "scores": torch.tensor([[-1.0, -2, -3, -4, -5, -6]], device="cuda")})
    assert search.done.tolist() == [1] and search.pool_scores.tolist() == [[-1, -2, -3]]


def test_start_of_single_sequences_leaves_the_others(bs):
    import torch
    from opentail.stingray_b200 import BeamSearch

    search = BeamSearch(6, 4, 5, eos=[2])
    for name in ("tokens", "parents", "steps", "done", "pool_steps", "pool_parents", "pool_tokens"):
        getattr(search, name).fill_(3)
    search.scores.fill_(-4.0)
    search.pool_scores.fill_(-5.0)
    bs.beam_start(search, 2, 3)
    torch.cuda.synchronize()
    assert search.steps.tolist() == [3, 3, 0, 0, 0, 3] and search.done.tolist() == [3, 3, 0, 0, 0, 3]
    assert search.scores[1].tolist() == [-4.0] * 4 and search.scores[2].tolist() == [0.0] + [-np.inf] * 3 and search.scores[5].tolist() == [-4.0] * 4
    assert search.pool_scores[1].tolist() == [-5.0] * 4 and search.pool_steps[4].tolist() == [-1] * 4
    assert search.parents[3].tolist() == [0, 1, 2, 3] and search.parents[5].tolist() == [3] * 4


def test_sequences_at_steps_of_their_own(bs):
    """A sequence that a new request takes over in the middle of the others writes its own rows of the trail."""
    import torch
    from opentail.stingray_b200 import BeamSearch

    rng = np.random.default_rng(5)
    B, K, n, T = 4, 3, 9, 7
    search = BeamSearch(B, K, T, eos=[2], length_penalty=0.5)
    norms = search.norms.cpu().tolist()
    bs.beam_start(search)
    rows = [beam_oracle.Search(K, T, [2], 0, norms) for _ in range(B)]
    for t in range(2 * T):
        if t == 3:
            bs.beam_start(search, 1, 2)
            rows[1], rows[2] = beam_oracle.Search(K, T, [2], 0, norms), beam_oracle.Search(K, T, [2], 0, norms)
        tok, par, sc = _candidates(rng, B, K, n, t, [], False)
        tok[tok == 5] = 2 if t % 5 == 4 else 6
        bs.beam_advance(search, {"tokens": torch.from_numpy(tok).cuda(), "parents": torch.from_numpy(par).cuda(), "scores": torch.from_numpy(sc).cuda()})
        for b, r in enumerate(rows):
            r.advance([(int(tok[b, i]), int(par[b, i]), sc[b, i]) for i in range(n)])
        _same(search, rows, T)


# ---- backtrace -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,B,K,N", [(1, 1, 1, 1), (2, 3, 4, 4), (37, 5, 3, 7), (300, 2, 8, 8), (1000, 3, 32, 32), (64, 64, 8, 8), (257, 1, 5, 128), (4099, 2, 4, 6),
                                     (20000, 1, 16, 3)])
def test_backtrace(bs, T, B, K, N):
    import torch

    rng = np.random.default_rng(T)
    tok, par = rng.integers(1, 1000, (T, B, K)).astype(np.int32), rng.integers(0, K, (T, B, K)).astype(np.int32)
    ends, first = rng.integers(0, T, (B, N)).astype(np.int32), rng.integers(0, K, (B, N)).astype(np.int32)
    last = rng.integers(1, 1000, (B, N)).astype(np.int32)
    ends[0, 0] = T - 1
    ends.reshape(-1)[1::5] = rng.choice([-1, T, -5, 0, T - 1], ends.reshape(-1)[1::5].shape)
    first.reshape(-1)[2::7] = rng.choice([-1, K, 1 << 30, -(1 << 31)], first.reshape(-1)[2::7].shape)
    if T > 30:  # trails that break off
        par[T // 3, 0, K // 2] = -1
        par[T // 2, B - 1, 0] = K
    out = {"sequences": torch.full((B, N, T), -77, dtype=torch.int32, device="cuda"), "lengths": torch.full((B, N), -77, dtype=torch.int32, device="cuda")}
    dev = [torch.from_numpy(v).cuda() for v in (tok, par, ends, first, last)]
    got = bs.beam_backtrace(*dev, pad=-3, out=out)
    seq, lengths = got["sequences"].cpu().numpy(), got["lengths"].cpu().numpy()
    for b in range(B):
        for i in range(N):
            row, length = beam_oracle.backtrace(tok[:, b], par[:, b], int(ends[b, i]), int(first[b, i]), int(last[b, i]), -3)
            assert lengths[b, i] == length and seq[b, i].tolist() == row, (b, i)


def test_backtrace_sequences_that_share_their_beginning(bs):
    import torch

    T, K = 90, 4
    tok = torch.arange(T * K, dtype=torch.int32).view(T, 1, K).cuda()
    par = torch.zeros((T, 1, K), dtype=torch.int32).cuda()
    same = torch.full((1, 4), T - 1, dtype=torch.int32, device="cuda")
    got = bs.beam_backtrace(tok, par, same, torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), same)["sequences"][0].cpu()
    for n in range(4):
        assert got[n].tolist() == [4 * t for t in range(T - 2)] + [4 * (T - 2) + n, T - 1]


def test_backtrace_into_wider_rows(bs):
    """out_stride: what lies behind n_steps is left alone; no lengths wanted."""
    import torch
    from opentail.stingray_b200 import _native as N

    lib, T, B, K = N.load(), 21, 2, 3
    g = torch.Generator().manual_seed(1)
    tok, par = torch.randint(0, 99, (T, B, K), generator=g, dtype=torch.int32).cuda(), torch.randint(0, K, (T, B, K), generator=g, dtype=torch.int32).cuda()
    ends = torch.full((B, K), T - 1, dtype=torch.int32, device="cuda")
    first = torch.zeros((B, K), dtype=torch.int32, device="cuda")
    want = bs.beam_backtrace(tok, par, ends, first, first)["sequences"]
    out = torch.full((B, K, T + 5), -8, dtype=torch.int32, device="cuda")
    rc = lib.stg_beam_backtrace(bs._h, tok.data_ptr(), par.data_ptr(), T, B, K, K, ends.data_ptr(), first.data_ptr(), first.data_ptr(), 0, out.data_ptr(), T + 5,
                                None, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(out[:, :, :T], want) and (out[:, :, T:] == -8).all()


# ---- reorder -------------------------------------------------------------------------------------------

def _parents(kind, B, K, rng):
    if kind == "same":
        p = np.tile(np.arange(K), (B, 1))
    elif kind == "one":
        p = np.full((B, K), K - 1)
    elif kind == "cycle":
        p = np.tile(np.roll(np.arange(K), 1), (B, 1))
    elif kind == "reverse":
        p = np.tile(np.arange(K)[::-1], (B, 1))
    else:
        p = rng.integers(0, K, (B, K))
        p[rng.random((B, K)) < 0.15] = rng.choice([-1, K, 1 << 30])
    return p.astype(np.int32).copy()


def _moved(t, parents, beam_dim, position_dim, positions):
    """What beam_reorder makes of `t` (CPU)."""
    import torch

    B, K = parents.shape
    t = t.movedim(beam_dim, 0)
    new = t.clone()
    pos = None if position_dim is None else position_dim % t.dim()
    if pos is not None:
        pos = pos + 1 if pos < beam_dim % t.dim() else pos  # the dimension after the move
    for b in range(B):
        for k in range(K):
            p = int(parents[b, k])
            if not 0 <= p < K:
                continue
            to, of = new[b * K + k], t[b * K + p]
            if pos is not None and positions is not None:
                used = min(max(int(positions[b]), 0), t.shape[pos])
                to, of = to.narrow(pos - 1, 0, used), of.narrow(pos - 1, 0, used)
            to.copy_(of)
    return torch.clone(new.movedim(0, beam_dim))


def _random(shape, dtype, seed):
    import torch

    g = torch.Generator().manual_seed(seed)
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g).to(dtype)
    return torch.randint(-100, 100, shape, generator=g).to(dtype)


def _layouts(R):
    """(shape, strides or None, dtype, beam_dim, position_dim)"""
    import torch

    return [
        ((R, 2, 40, 16), None, torch.bfloat16, 0, 2),
        ((R, 2, 16, 41), None, torch.bfloat16, 0, 3),       # positions innermost, odd
        ((R, 40, 2, 8), None, torch.float32, 0, 1),
        ((3, R, 2, 10, 4), None, torch.float16, 1, 3),      # layers in front of the beams
        ((2, 2, R, 5, 3), None, torch.float32, 2, 3),
        ((R, 7), None, torch.int32, 0, 1),                  # a page table
        ((R,), None, torch.int64, 0, None),
        ((R, 3), None, torch.uint8, 0, None),
        ((R, 1000), None, torch.int8, 0, 1),
        ((R, 33, 5), None, torch.float32, 0, None),
        ((R, 12, 6), (100, 8, 1), torch.float32, 0, 1),     # gaps inside a row: positions are an outer dimension
        ((R, 4, 9, 6), (600, 140, 12, 2), torch.int16, 0, 2),  # every other element
        ((6, R), None, torch.float64, 1, 0),                # beams innermost
        ((R, 300), (301, 1), torch.bfloat16, 0, 1),         # rows at odd addresses
        ((R, 1, 5), None, torch.float32, 0, 1),             # one position
    ]


@pytest.mark.parametrize("B,K", [(1, 1), (1, 2), (3, 4), (2, 5), (4, 8), (2, 13), (3, 16), (2, 32)])
@pytest.mark.parametrize("kind", ["random", "one", "cycle", "reverse", "same"])
def test_reorder_layouts(bs, B, K, kind):
    import torch
    from opentail.stingray_b200 import BeamStates

    rng = np.random.default_rng(K)
    parents = _parents(kind, B, K, rng)
    dev_parents = torch.from_numpy(parents).cuda()
    R = B * K
    for positions in (None, 3, "each"):
        tensors, before, dims = [], [], []
        for i, (shape, strides, dtype, beam_dim, pos) in enumerate(_layouts(R)):
            x = _random(shape, dtype, i)
            if strides is None:
                t = x.cuda()
                whole = t
            else:  # in a buffer whose other bytes must not change
                span = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
                whole = torch.full((span + 7,), 55, dtype=dtype, device="cuda")
                t = torch.as_strided(whole, shape, strides, 0)
                t.copy_(x)
            tensors.append((t, whole, whole.cpu().clone(), beam_dim, pos))
        each = rng.integers(-1, 45, B).astype(np.int32)
        given = torch.from_numpy(each).cuda() if positions == "each" else positions
        used = each if positions == "each" else None if positions is None else [positions] * B
        for t, whole, old, beam_dim, pos in tensors:
            x = t.cpu().clone()
            bs.beam_reorder(BeamStates([t], K, beam_dim=beam_dim, position_dim=pos), dev_parents, positions=given)
            assert torch.equal(t.cpu(), _moved(x, parents, beam_dim, pos, used)), (tuple(t.shape), t.stride(), positions)
            if whole is not t:  # the gaps
                now = whole.cpu()
                torch.as_strided(now, t.shape, t.stride(), 0).fill_(1)
                torch.as_strided(old, t.shape, t.stride(), 0).fill_(1)
                assert torch.equal(now, old)


@pytest.mark.parametrize("K", [1, 2, 3])
@pytest.mark.parametrize("kind", ["random", "one", "reverse"])
def test_reorder_of_runs_of_several_tiles(bs, K, kind):
    """Two columns to a thread of two beams, one of three: whole tiles, tiles that end within a run, runs that end within a vector."""
    import torch
    from opentail.stingray_b200 import BeamStates

    B = 5
    rng = np.random.default_rng(K + 10)
    parents = _parents(kind, B, K, rng)
    R = B * K
    for shape, strides, dtype, pos in [((R, 2, 700, 80), None, torch.bfloat16, 2), ((R, 3, 500, 33), None, torch.float32, 2),
                                       ((R, 5, 16, 1001), None, torch.bfloat16, 3), ((R, 40000), (40003, 1), torch.bfloat16, 1),
                                       ((R, 8192), None, torch.float32, 1), ((R, 2, 4100, 4), (32816, 16404, 4, 1), torch.float32, 2),
                                       ((R, 50000), (50001, 1), torch.uint8, 1)]:
        x = _random(shape, dtype, K)
        t = x.cuda() if strides is None else torch.as_strided(torch.zeros(R * strides[0] + 1, dtype=dtype, device="cuda"), shape, strides, 1).copy_(x)
        room = shape[pos]
        for used in (None, np.full(B, room - 1), rng.integers(0, room + 2, B)):
            given = None if used is None else torch.from_numpy(used.astype(np.int32)).cuda()
            want = _moved(t.cpu(), parents, 0, pos, used)
            bs.beam_reorder(BeamStates([t], K, position_dim=pos), torch.from_numpy(parents).cuda(), positions=given)
            assert torch.equal(t.cpu(), want), (shape, strides, used)


def test_reorder_many_states_of_all_sizes_at_once(bs):
    """More states than one launch takes; some empty, some shared out over many tiles."""
    import torch
    from opentail.stingray_b200 import BeamStates

    rng = np.random.default_rng(3)
    B, K = 5, 4
    parents = _parents("random", B, K, rng)
    xs = [_random((B * K, int(rng.integers(0, 4)), int(rng.integers(1, 900)), int(rng.integers(1, 40))), torch.bfloat16, i) for i in range(110)]
    ts = [x.cuda() for x in xs]
    bs.beam_reorder(BeamStates(ts, K, position_dim=2), torch.from_numpy(parents).cuda(), positions=500)
    for t, x in zip(ts, xs):
        assert torch.equal(t.cpu(), _moved(x, parents, 0, 2, [500] * B))


def test_reorder_leaves_rows_behind_the_last_sequence(bs):
    import torch
    from opentail.stingray_b200 import BeamStates

    x = _random((24, 4, 50, 8), torch.bfloat16, 1)
    t = x.cuda()
    parents = _parents("cycle", 4, 4, None)
    bs.beam_reorder(BeamStates([t[:16]], 4, position_dim=2), torch.from_numpy(parents).cuda(), positions=50)
    assert torch.equal(t[16:].cpu(), x[16:]) and torch.equal(t[:16].cpu(), _moved(x[:16], parents, 0, 2, [50] * 4))


def test_reorder_of_a_large_cache(bs):
    """Offsets within a row and between rows that pass 32 bits."""
    import torch
    from opentail.stingray_b200 import BeamStates

    K, S = 4, 9 << 20
    t = torch.empty((K, S, 64), dtype=torch.bfloat16, device="cuda")  # 1.2 GB a row
    for k in range(K):
        t[k] = k + 1
    t[:, -1] = t[:, -1] * 10
    parents = torch.tensor([[2, 2, 0, 1]], dtype=torch.int32, device="cuda")
    bs.beam_reorder(BeamStates([t], K, position_dim=1), parents, positions=S - 1)
    for k, p in enumerate([2, 2, 0, 1]):
        assert bool((t[k, :-1] == p + 1).all()) and bool((t[k, -1] == 10 * (k + 1)).all())
    bs.beam_reorder(BeamStates([t], K, position_dim=1), parents)
    assert t[:, -1, 0].tolist() == [30.0, 30.0, 10.0, 20.0] and t[:, 0, 0].tolist() == [1.0, 1.0, 3.0, 3.0]


def test_reorder_of_the_handles_histories(bs):
    """The histories follow their beams: sampling with penalties sees the parent's tokens."""
    import torch
    from opentail.stingray_b200 import BeamStates, SamplingParams

    rng = np.random.default_rng(3)
    B, K, V = 3, 4, 500
    R = B * K
    hist = [rng.integers(0, V, n).astype(np.int32) for n in np.repeat([0, 5, 40], K)]
    bs.history_reset()
    for r in range(R):
        bs.history_load(r, hist[r])
    parents = _parents("random", B, K, rng)
    state = _random((R, 5), torch.float32, 1)
    t = state.cuda()
    bs.beam_reorder(BeamStates([t], K), torch.from_numpy(parents).cuda(), history=True)
    want = list(hist)
    for b in range(B):
        for k in range(K):
            if 0 <= parents[b, k] < K:
                want[b * K + k] = hist[b * K + parents[b, k]]
    x = torch.from_numpy(rng.normal(0, 1, (R, V)).astype(np.float32)).cuda()
    params = [SamplingParams(Temperature=0.0, PresencePenalty=3.0, FrequencyPenalty=0.5, RepeatLastN=0)] * R
    got = bs.sample_rows(x, params, history_ring=True)["tokens"]
    ids, off = np.concatenate(want), np.concatenate([[0], np.cumsum([len(w) for w in want])]).astype(np.int32)
    ref = bs.sample_rows(x, params, history_ids=torch.from_numpy(ids).cuda(), history_offsets=off)["tokens"]
    assert torch.equal(got, ref) and torch.equal(t.cpu(), _moved(state, parents, 0, None, None))
    # another length in one beam: refused, and nothing moves
    from opentail.stingray_b200 import StingrayError

    bs.history_load(5, hist[5][:3])
    kept = t.clone()
    with pytest.raises(StingrayError, match="differ in length"):
        bs.beam_reorder(BeamStates([t], K), torch.from_numpy(parents).cuda(), history=True)
    assert torch.equal(t, kept)
    bs.history_reset()


def _sampled_with(bs, hist, V, seed):
    """Greedy tokens of random rows whose penalties see the handle's histories, and the same with `hist` handed over."""
    import torch
    from opentail.stingray_b200 import SamplingParams

    x = torch.from_numpy(np.random.default_rng(seed).normal(0, 1, (len(hist), V)).astype(np.float32)).cuda()
    params = [SamplingParams(Temperature=0.0, PresencePenalty=3.0, FrequencyPenalty=0.5, RepeatLastN=0)] * len(hist)
    got = bs.sample_rows(x, params, history_ring=True)["tokens"]
    ids, off = np.array([t for h in hist for t in h], np.int32), np.concatenate([[0], np.cumsum([len(h) for h in hist])]).astype(np.int32)
    return got, bs.sample_rows(x, params, history_ids=torch.from_numpy(ids).cuda(), history_offsets=off)["tokens"]


def test_a_captured_reorder_moves_histories_of_the_replays_length(bs):
    """Captured while the histories are empty, replayed while direct appends make them longer."""
    import torch
    from opentail.stingray_b200 import BeamSearch

    B, K, V, T = 3, 4, 30, 25
    R = B * K
    g = torch.Generator().manual_seed(4)
    search = BeamSearch(B, K, T, eos=[2])
    x = torch.zeros((R, V), device="cuda")
    best = bs.beam_select(x, search.scores, search.n_candidates)
    bs.history_reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bs.beam_select(x, search.scores, search.n_candidates, out=best)
        bs.beam_advance(search, best)
        bs.beam_reorder(None, search.parents, history=True)
    bs.beam_start(search)
    hist = [[] for _ in range(R)]
    moved = 0
    for t in range(T):
        x.copy_(torch.randn((R, V), generator=g) * 2)
        graph.replay()
        parents, tokens = search.parents.tolist(), search.tokens.flatten().tolist()
        hist = [hist[b * K + parents[b][k]] + [tokens[b * K + k]] for b in range(B) for k in range(K)]
        moved += sum(p != k for row in parents for k, p in enumerate(row))
        bs.history_append(search.tokens.flatten())
        if t % 8 == 7 or t == T - 1:
            got, want = _sampled_with(bs, hist, V, t)
            assert torch.equal(got, want), t
    assert moved > T
    # a direct call behind the replays
    parents = _parents("reverse", B, K, None)
    bs.beam_reorder(None, torch.from_numpy(parents).cuda(), history=True)
    got, want = _sampled_with(bs, [hist[b * K + parents[b, k]] for b in range(B) for k in range(K)], V, 77)
    assert torch.equal(got, want)
    bs.history_reset()


def test_a_replayed_reorder_leaves_histories_of_different_lengths(bs):
    """What a direct call refuses: the sequence whose beams differ stays as it is, the others move."""
    import torch

    rng = np.random.default_rng(8)
    B, K, V = 3, 4, 300
    parents = _parents("cycle", B, K, None)
    dev = torch.from_numpy(parents).cuda()
    bs.history_reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bs.beam_reorder(None, dev, history=True)
    hist = [rng.integers(0, V, n).tolist() for n in [7] * 4 + [7, 9, 7, 7] + [30] * 4]
    for r, h in enumerate(hist):
        bs.history_load(r, np.array(h, np.int32))
    graph.replay()
    want = [hist[b * K + (k if b == 1 else parents[b, k])] for b in range(B) for k in range(K)]
    got, ref = _sampled_with(bs, want, V, 1)
    assert torch.equal(got, ref)
    bs.history_reset()


def test_histories_that_move_on_another_stream(bs):
    """The handle's calls are put one behind the other: a step on one stream samples before, or behind, a reordering on another."""
    import torch
    from opentail.stingray_b200 import SamplingParams

    rng = np.random.default_rng(2)
    B, K, V = 2, 4, 400
    R = B * K
    parents = _parents("reverse", B, K, None)
    dev = torch.from_numpy(parents).cuda()
    hist = [rng.integers(0, V, 30).astype(np.int32) for _ in range(R)]
    after = [hist[b * K + parents[b, k]] for b in range(B) for k in range(K)]
    x = torch.from_numpy(rng.normal(0, 1, (R, V)).astype(np.float32)).cuda()
    params = [SamplingParams(Temperature=0.0, PresencePenalty=3.0, FrequencyPenalty=0.5, RepeatLastN=0)] * R

    def sampled(h):
        ids, off = np.concatenate(h), np.arange(R + 1, dtype=np.int32) * 30
        return bs.sample_rows(x, params, history_ids=torch.from_numpy(ids).cuda(), history_offsets=off)["tokens"]

    want = [sampled(hist), sampled(after)]
    assert not torch.equal(*want)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for first_moves in (False, True):
        for r in range(R):
            bs.history_load(r, hist[r])
        torch.cuda.synchronize()
        out = torch.full((R,), -1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            torch.cuda._sleep(40_000_000)  # some 20 ms
            if first_moves:
                bs.beam_reorder(None, dev, history=True)
            else:
                bs.sample_rows(x, params, history_ring=True, out={"tokens": out})
        with torch.cuda.stream(two):
            if first_moves:
                bs.sample_rows(x, params, history_ring=True, out={"tokens": out})
            else:
                bs.beam_reorder(None, dev, history=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want[1 if first_moves else 0])
    bs.history_reset()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("B,K", [(4, 2), (3, 5), (2, 20)])
def test_histories_move_whatever_positions_the_states_have_in_use(bs, B, K, captured):
    """The positions are the states'; a history goes by its own length."""
    import torch
    from opentail.stingray_b200 import BeamStates

    rng = np.random.default_rng(K)
    R, V = B * K, 300
    hist = [rng.integers(0, V, n).tolist() for n in np.repeat(rng.integers(1, 41, B), K)]
    parents = _parents("random", B, K, rng)
    dev = torch.from_numpy(parents).cuda()
    x = _random((R, 3, 12, 5), torch.float32, K)
    each = torch.from_numpy(rng.integers(0, 14, B).astype(np.int32)).cuda()
    for positions in (None, 0, 3, each):
        bs.history_reset()
        t = x.cuda()
        states = BeamStates([t], K, position_dim=2)
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                bs.beam_reorder(states, dev, positions=positions, history=True)
        for r, h in enumerate(hist):
            bs.history_load(r, np.array(h, np.int32))
        if captured:
            graph.replay()
        else:
            bs.beam_reorder(states, dev, positions=positions, history=True)
        want = [hist[b * K + (p if 0 <= (p := parents[b, k]) < K else k)] for b in range(B) for k in range(K)]
        got, ref = _sampled_with(bs, want, V, K)
        assert torch.equal(got, ref), positions
        used = None if positions is None else each.tolist() if positions is each else [positions] * B
        assert torch.equal(t.cpu(), _moved(x, parents, 0, 2, used))
    bs.history_reset()


def test_refusals(bs):
    import ctypes as C

    import torch
    from opentail.stingray_b200 import BeamSearch, BeamStates, StingrayError
    from opentail.stingray_b200 import _native as N

    par = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    t = torch.zeros((8, 16), device="cuda")
    with pytest.raises(ValueError):
        BeamStates([t], 3)
    with pytest.raises(ValueError):
        BeamStates([t.cpu()], 4)
    with pytest.raises(ValueError):
        BeamStates([t], 4, position_dim=0)
    with pytest.raises(ValueError):
        BeamStates([torch.zeros((8, 4, 4, 4, 4, 4), device="cuda")[:, ::2, ::2, ::2, ::2, ::2]], 4)
    with pytest.raises(StingrayError, match="overlap"):
        bs.beam_reorder(BeamStates([torch.zeros(16, device="cuda").expand(8, 16)], 4), par)
    with pytest.raises(StingrayError, match="overlap"):
        bs.beam_reorder(BeamStates([torch.as_strided(torch.zeros(100, device="cuda"), (8, 16), (8, 1))], 4), par)
    with pytest.raises(ValueError):
        bs.beam_reorder(BeamStates([t], 4), par[:1])
    with pytest.raises(ValueError):
        bs.beam_reorder(BeamStates([t], 4), par.long())
    with pytest.raises(ValueError):
        bs.beam_reorder(BeamStates([t], 4), par, positions=-1)
    with pytest.raises(StingrayError, match="max_rows"):
        bs.beam_reorder(None, torch.zeros((129, 4), dtype=torch.int32, device="cuda"))
    r = N.StgBeamReorder(C.sizeof(N.StgBeamReorder), 2, 4, 0, None, par.data_ptr(), None, -1, 1)
    assert bs._lib.stg_beam_reorder(bs._h, C.byref(r), None) == 1  # unknown flag
    r = N.StgBeamReorder(C.sizeof(N.StgBeamReorder), 2, 4, 0, None, par.data_ptr() + 2, None, -1, 0)
    assert bs._lib.stg_beam_reorder(bs._h, C.byref(r), None) == 1  # misaligned
    with pytest.raises(ValueError):
        BeamSearch(1, 33, 4)
    with pytest.raises(ValueError):
        BeamSearch(1, 4, 0)
    with pytest.raises(ValueError):
        BeamSearch(1, 4, 4, eos=list(range(9)))
    search = BeamSearch(2, 4, 3, eos=[2])
    with pytest.raises(StingrayError):
        bs.beam_start(search, 1, 2)
    c = {"tokens": par, "parents": par, "scores": torch.zeros((2, 4), device="cuda")}
    with pytest.raises(ValueError):
        bs.beam_advance(search, {**c, "scores": c["scores"].double()})
    with pytest.raises(ValueError):
        bs.beam_advance(search, {k: v[:1].contiguous() for k, v in c.items()})
    with pytest.raises(StingrayError, match="128"):
        bs.beam_advance(search, {k: v.repeat(1, 33) for k, v in c.items()})
    trail = torch.zeros((3, 2, 4), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        bs.beam_backtrace(trail, trail[:2], par, par, par)
    with pytest.raises(StingrayError, match="128"):
        wide = torch.zeros((2, 129), dtype=torch.int32, device="cuda")
        bs.beam_backtrace(trail, trail, wide, wide, wide)


# ---- together ------------------------------------------------------------------------------------------

def _decode(bs, B, K, V, T, eos, seed, capture):
    """A little model - the next token's logits depend on the token and on a state that the beam carries along - decoded
    with the library, and the same search in plain Python."""
    import torch
    from opentail.stingray_b200 import BeamSearch, BeamStates

    g = torch.Generator().manual_seed(seed)
    table = (torch.randn((V, V), generator=g) * 2).cuda()
    drift = torch.randn((V, 8), generator=g).cuda()
    head = (torch.randn((8, V), generator=g) * 0.5).cuda()
    start = torch.randn((B, 8), generator=g).cuda()
    search = BeamSearch(B, K, T, eos=eos, length_penalty=0.8)
    state = start.repeat_interleave(K, 0).contiguous()
    path = torch.full((B * K, T), -1, dtype=torch.int32, device="cuda")  # a cache: what the beam has taken
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    used = torch.zeros(B, dtype=torch.int32, device="cuda")
    states = BeamStates([state, path], K, position_dim=[None, 1])
    bs.beam_start(search)
    best = bs.beam_select(torch.zeros((B * K, V), device="cuda"), search.scores, search.n_candidates)

    def one():
        logits = table[search.tokens.flatten().long()] + state @ head
        bs.beam_select(logits, search.scores, search.n_candidates, out=best)
        bs.beam_advance(search, best)
        bs.beam_reorder(states, search.parents, positions=used)
        state.copy_(state * 0.5 + drift[search.tokens.flatten().long()])
        path.index_copy_(1, step, search.tokens.view(-1, 1))
        step.add_(1)
        used.add_(1)
        return logits

    if capture:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        kept = [v.clone() for v in (state, path, step, used)]
        with torch.cuda.stream(side):
            one()  # warm
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = one()
        for v, k in zip((state, path, step, used), kept):
            v.copy_(k)
        bs.beam_start(search)
    seen = []
    for t in range(T):
        if capture:
            graph.replay()
            seen.append(logits.clone())
        else:
            seen.append(one())
    found = bs.beam_backtrace(search.trail_tokens, search.trail_parents, search.pool_steps, search.pool_parents, search.pool_tokens)
    # the same in Python, on the logits that the steps saw
    norms = search.norms.cpu().tolist()
    rows = [beam_oracle.Search(K, T, eos, 0, norms) for _ in range(B)]
    texts = [[[] for _ in range(K)] for _ in range(B)]
    ended = [[] for _ in range(B)]
    for t in range(T):
        x = seen[t].cpu().numpy().reshape(B, K, V)
        for b, r in enumerate(rows):
            if r.done:
                continue
            s = np.array([[v[2] for v in r.beams]], np.float32)
            cand = beam_oracle.select(x[b], s, search.n_candidates)[0][0]
            before, old = texts[b], list(r.pool)
            r.advance([(v, k, np.float32(sc)) for sc, k, v, _ in cand])
            for e in r.pool:
                if e not in old:
                    ended[b].append((e, before[e[2]] + [e[3]]))
            texts[b] = [before[p] + [tok] for tok, p in r.trail[-1]]
    for b, r in enumerate(rows):
        assert int(search.steps[b]) == r.steps and bool(search.done[b]) == r.done
        assert search.pool_tokens[b, :len(r.pool)].tolist() == [e[3] for e in r.pool]
        # per step a row's normaliser is off by at most 2.3e-6 (tests/test_gpu_beam_select.py) and both sides round once
        assert np.allclose(search.pool_scores[b, :len(r.pool)].cpu().numpy(), [e[0] for e in r.pool], rtol=T * 2.0 ** -23, atol=T * 2.3e-6)
        for i, e in enumerate(r.pool):
            text = next(tx for en, tx in ended[b] if en == e)
            n = int(found["lengths"][b, i])
            assert n == e[1] + 1 and found["sequences"][b, i, :n].tolist() == text
    return path, search


def test_kernels_behind_one_another_wait_for_one_another(bs):
    """Each kernel starts while the one ahead of it ends: a chain without a pause gives what it gives with one behind every call."""
    import torch
    from opentail.stingray_b200 import BeamSearch, BeamStates

    def chain(pause):
        g = torch.Generator().manual_seed(9)
        B, K, V, T = 16, 4, 4001, 60
        logits = torch.randn((T, B * K, V), generator=g).cuda() * 2
        state = torch.randn((B * K, 3, 37), generator=g).cuda()
        search = BeamSearch(B, K, T, eos=[1, 2], length_penalty=0.9)
        states = BeamStates([state], K)
        bs.beam_start(search)
        pause()
        best = None
        for t in range(T):
            best = bs.beam_select(logits[t], search.scores, search.n_candidates, out=best)
            pause()
            bs.beam_advance(search, best)
            pause()
            bs.beam_reorder(states, search.parents)
            pause()
        found = bs.beam_backtrace(search.trail_tokens, search.trail_parents, search.pool_steps, search.pool_parents, search.pool_tokens)
        return [state, search.pool_scores, search.steps, found["sequences"], found["lengths"]]

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        for a, b in zip(chain(lambda: None), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("capture", [False, True])
@pytest.mark.parametrize("B,K,V,T,eos", [(1, 4, 97, 12, [2]), (5, 3, 201, 9, [2, 7]), (3, 8, 64, 20, []), (2, 1, 50, 6, [1])])
def test_a_whole_search(bs, B, K, V, T, eos, capture):
    import torch

    path, search = _decode(bs, B, K, V, T, eos, 10 * B + K, capture)
    if not eos:  # the beams' caches hold what the trail says they took, up to the last reordering
        ends = torch.full((B, K), T - 1, dtype=torch.int32, device="cuda")
        own = bs.beam_backtrace(search.trail_tokens, search.trail_parents, ends, search.trail_parents[-1].contiguous(), search.trail_tokens[-1].contiguous())
        best = own["sequences"].view(B * K, T)[:, :T - 2]
        assert {tuple(r) for r in best.tolist()} <= {tuple(r) for r in path[:, :T - 2].tolist()}
