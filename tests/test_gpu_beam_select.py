"""stg_beam_select against the definition in 64 bits.

Tolerances.  The sum S of a row's terms 2^(x log2(e) - c) is made of fp32 terms: the exponential is off by at most 2^-22 of a
term; its argument is rounded twice, by 2^-24 of its size, which is at most 5 for the largest terms and of no account for the small
ones (d * 2^-d < 0.54): 2 * 5 * 0.7 * 2^-24; and at most 32 terms are added up in 32 bits before 64 take over, 31 * 2^-24.  Together
below 2.3e-6 of S, which is what log S and every score of the row may be off by (LSE); a score is rounded to 32 bits once more.
So two candidates of different beams may change places only if their scores lie within 2 * LSE; candidates of one beam never."""
import numpy as np
import pytest

from tests import beam_oracle

pytestmark = pytest.mark.gpu
LSE = 2.3e-6


def _sampler(**kw):
    from opentail.stingray_b200 import BatchSampler

    return BatchSampler(**{"max_rows": 64, "max_vocab": 262144, "max_history": 8, "max_top_k": 8, **kw})


@pytest.fixture(scope="module")
def bs():
    b = _sampler()
    yield b
    b.close()


def _words(allowed):
    rows, vocab = allowed.shape
    bits = np.zeros((rows, (vocab + 31) // 32 * 32), bool)
    bits[:, :vocab] = allowed
    return np.packbits(bits.reshape(rows, -1, 32), axis=-1, bitorder="little").view(np.uint32).reshape(rows, -1).view(np.int32)


def _check(bs, x, scores, n, *, allowed=None, uses=None, garbage=None, softcap=0.0, stride=None, shift=0):
    """x: torch CPU tensor [B * K, V].  `stride`, `shift`: laid out in a wider buffer, starting `shift` elements in."""
    import torch

    rows, vocab = x.shape
    scores = np.asarray(scores, np.float32)
    B, K = scores.shape
    if garbage is not None:  # what masked places hold
        x = torch.where(torch.from_numpy(allowed), x, torch.tensor(garbage, dtype=x.dtype))
    stride = stride or vocab
    buf = torch.full((shift + rows * stride,), float("nan"), dtype=x.dtype, device="cuda")
    view = buf[shift:].view(rows, stride)[:, :vocab]
    view.copy_(x)
    mask = None if allowed is None else torch.from_numpy(_words(allowed)).cuda()
    use = None if uses is None else torch.from_numpy(np.asarray(uses, np.uint8)).cuda()
    got = bs.beam_select(view, torch.from_numpy(scores).cuda(), n, mask=mask, row_uses_mask=use, softcap=softcap, want_norms=True, want_flags=True)
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in got.items()}
    read = view.float()
    if softcap:
        read = torch.tanh(read / torch.full_like(read, softcap)) * softcap  # a division by a number would be a product
    read = read.cpu().numpy().astype(np.float64)
    if allowed is not None:
        on = allowed if uses is None else allowed | (np.asarray(uses)[:, None] == 0)
        read = np.where(on, read, -np.inf)
    want, norms = beam_oracle.select(read, scores, min(n, K * vocab))
    for b in range(B):
        place = {(k, v): s for s, k, v, _ in beam_oracle.select(read[b * K:(b + 1) * K], scores[b:b + 1], n + 8)[0][0]}
        assert (got["flags"][b] & 1 != 0) == (len(want[b]) < n)
        bad = any(np.isfinite(scores[b, k]) and np.isnan(norms[b, k]) for k in range(K))
        empty = any(np.isfinite(scores[b, k]) and norms[b, k] == -np.inf for k in range(K))
        assert (got["flags"][b] & 2 != 0) == bad and (got["flags"][b] & 64 != 0) == empty
        last = {}
        seen = set()
        for i in range(n):
            tok, par, sc = int(got["tokens"][b, i]), int(got["parents"][b, i]), got["scores"][b, i]
            if i >= len(want[b]):
                assert (tok, par, sc) == (-1, -1, -np.inf)
                continue
            s, k, v, _ = want[b][i]
            if (par, tok) != (k, v):
                assert par != k and (par, tok) in place and abs(place[par, tok] - s) <= 2 * LSE, (b, i, (par, tok), (k, v))
            assert abs(float(sc) - s) <= 2 * LSE + abs(s) * 2.0 ** -24 + LSE, (b, i, float(sc), s)
            assert (par, tok) not in seen
            seen.add((par, tok))
            value = read[b * K + par, tok]
            assert par not in last or (-value, tok) > last[par]  # within a beam: the larger logit, then the lower token
            last[par] = (-value, tok)
        for k in range(K):
            if np.isnan(norms[b, k]):
                assert not np.isfinite(got["log_norms"][b, k])
            elif norms[b, k] == -np.inf:
                assert got["log_norms"][b, k] == -np.inf
            else:
                assert abs(got["log_norms"][b, k] - norms[b, k]) <= LSE + abs(norms[b, k]) * 2.0 ** -24
    return got


def _normal(rows, vocab, seed, dtype="f32", scale=3.0):
    import torch

    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g) * scale
    return x.to(torch.bfloat16) if dtype == "bf16" else x


def _scores(B, K, seed):
    return -np.cumsum(np.random.default_rng(seed).random((B, K)) * 3, 1).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 1, 1, 3), (2, 3, 2, 6), (3, 4, 5, 20), (1, 2, 31, 4), (2, 2, 33, 128), (1, 32, 7, 64),
                                     (2, 32, 300, 128), (5, 1, 257, 2), (3, 4, 4095, 8), (3, 4, 4096, 8), (2, 4, 4097, 8), (2, 3, 8192, 9),
                                     (2, 2, 8193, 16), (2, 5, 16391, 13), (1, 4, 50257, 8), (4, 4, 65536, 8), (1, 7, 151936, 21), (2, 2, 262144, 4)])
def test_sizes(bs, B, K, V, n, dtype):
    _check(bs, _normal(B * K, V, V + K, dtype), _scores(B, K, V), n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("stride,shift", [(20016, 0), (20013, 0), (20016, 1), (20016, 4), (20024, 8), (20012, 2)])
def test_strides_and_offsets(bs, dtype, stride, shift):
    _check(bs, _normal(6, 20011, 5, dtype), _scores(2, 3, 1), 7, stride=stride, shift=shift)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 1000, 20011, 70000])
def test_equal_logits_go_to_the_lower_token(bs, V, dtype):
    """Rows of one value, of few values, and of one value with few above it."""
    import torch

    x = torch.zeros((6, V))
    x[1] = 2.5
    g = torch.Generator().manual_seed(V)
    x[2] = torch.randint(-2, 2, (V,), generator=g).float()
    x[3] = torch.where(torch.rand(V, generator=g) < 0.01, 1.0, 0.0)
    x[4] = -0.0
    x[4, ::3] = 0.0
    x[5, V // 2:] = 1.0
    x = x.to(torch.bfloat16) if dtype == "bf16" else x
    _check(bs, x, _scores(2, 3, V), 40)
    _check(bs, x, _scores(6, 1, V), 128)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_of_any_size(bs, dtype):
    """Rows far from zero, rows that grow along the vocabulary, logits next to and beyond 1e6, and mixtures of all of them."""
    import torch

    V = 40000
    x = _normal(16, V, 21)
    for r, shift in enumerate((300.0, -300.0, 5000.0, -5000.0, 999990.0, -999990.0, 1e6, -1e6, 1.5e6, -1.5e6, 3e7, -3e7)):
        x[r] = x[r] * (0.01 if abs(shift) > 1e5 else 1.0) + shift
    x[12] += torch.arange(V) * 0.02                      # 800 from one end to the other
    x[13] -= torch.arange(V) * 0.02
    x[14, ::5000] = torch.tensor([1e6, -1e6, 2e6, 999999.0, -3e6, 1000001.0, 5.0, 2000003.0])
    x[15, 700:20000] = torch.finfo(torch.float32).min
    x[15, 20000:] -= 1e6
    x = x.to(torch.bfloat16) if dtype == "bf16" else x
    _check(bs, x, _scores(16, 1, 5), 20)
    _check(bs, x, _scores(4, 4, 5), 20)
    _check(bs, x.flip(1), _scores(8, 2, 5), 9)
    _check(bs, x[:, :39990], _scores(16, 1, 5), 20, stride=40001)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("K,V,n", [(8, 39168, 24), (8, 39168, 38), (8, 39168, 40), (8, 20011, 20), (8, 20011, 41), (4, 65536, 63), (4, 65536, 65),
                                   (3, 131072, 128), (2, 8192, 7), (2, 8192, 9)])
def test_one_beam_far_ahead(bs, K, V, n, dtype):
    """All candidates come from one beam, which has about as many groups as there are candidates, or fewer: bounds out of
    the other beams' groups keep nothing away."""
    for masked in (False, True):
        scores = _scores(3, K, n) - 60.0
        scores[0, 0] += 60.0
        scores[1, K - 1] += 60.0
        scores[2] += 60.0
        scores[2, 1:] = -np.inf
        allowed = np.random.default_rng(n).random((3 * K, V)) < 0.3 if masked else None
        _check(bs, _normal(3 * K, V, n, dtype), scores, n, allowed=allowed, uses=np.arange(3 * K) % 3 != 1 if masked else None)
    for cap in (2.0, 30.0):
        _check(bs, _normal(3 * K, V, n, dtype) - (0.0 if cap > 2.0 else 20.0), scores, n, softcap=cap)


@pytest.mark.parametrize("V", [4096, 20011, 100000])
def test_rows_that_ascend_and_descend(bs, V):
    import torch

    up = torch.arange(V).float() * 0.001
    x = torch.stack([up, up.flip(0), up.view(-1).roll(V // 3), -up])
    for n in (4, 33, 128):
        _check(bs, x, _scores(2, 2, 3), n)


def test_best_logits_in_one_place(bs):
    """All of a row's best in one thread's share, in neighbouring tokens, at the ends."""
    import torch

    x = _normal(4, 30000, 9)
    x[0, :64] = 20 + torch.arange(64) * 0.01
    x[1, -64:] = 20 + torch.arange(64) * 0.01
    x[2, 1000:30000:1024] = 25.0
    x[3, 5:30000:256] = 25.0
    for n in (8, 64, 128):
        _check(bs, x, _scores(1, 4, 3), n)
        _check(bs, x, _scores(4, 1, 3), n)


def test_dead_beams(bs):
    x = _normal(12, 5000, 2)
    s = _scores(3, 4, 2)
    s[0, 1:] = -np.inf          # a first step
    s[1, :] = -np.inf           # a sequence that has ended
    s[2, 0], s[2, 1], s[2, 2] = np.nan, np.inf, -np.inf
    x[4:8] = float("nan")       # rows of dead beams hold anything
    got = _check(bs, x, s, 8)
    assert (got["tokens"][1] == -1).all() and (got["flags"][1] & 1) == 1


def test_rows_without_a_usable_normaliser(bs):
    x = _normal(12, 9000, 4)
    x[0, 17] = float("nan")
    x[1, 8999] = float("inf")
    x[2] = float("-inf")
    x[3, 4] = float("-inf")     # one -infinity is nothing special
    x[4] = float("nan")
    x[5:8] = float("-inf")
    x[8, :8999] = float("-inf")  # one token alone
    _check(bs, x, _scores(3, 4, 4), 16)


def test_lowest_values(bs):
    """The type's lowest value is a logit like any other."""
    import torch

    low = torch.finfo(torch.float32).min
    x = _normal(6, 6000, 4)
    x[0, 100:] = low
    x[1] = low
    x[2] = low
    x[2, 5] = 3.0
    x[3, :] = torch.finfo(torch.float32).max
    x[4, 7] = torch.finfo(torch.float32).max
    got = _check(bs, x[:3], _scores(1, 3, 4), 120)
    assert (got["tokens"] >= 0).all()
    _check(bs, x[3:], _scores(3, 1, 4), 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [31, 4097, 20011, 65536])
@pytest.mark.parametrize("garbage", [None, float("nan"), float("inf"), float("-inf")])
def test_masks(bs, V, dtype, garbage):
    rng = np.random.default_rng(V)
    dens = np.array([[0.0], [0.001], [0.02], [0.3], [0.9], [1.0], [0.0], [0.5]])
    allowed = rng.random((8, V)) < dens
    allowed[6, V - 1] = True
    _check(bs, _normal(8, V, 3, dtype), _scores(2, 4, 4), 9, allowed=allowed, garbage=garbage)
    _check(bs, _normal(8, V, 3, dtype), _scores(4, 2, 4), 9, allowed=allowed, uses=[1, 0, 1, 1, 0, 1, 1, 0])


@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("V,stride,shift", [(20010, 20010, 0), (20011, 20014, 0), (20010, 20014, 1), (20011, 20011, 1), (4098, 4098, 2), (1023, 1026, 0)])
def test_masked_rows_of_pairs(bs, V, stride, shift, softcap):
    """bf16 rows that begin at 4 bytes but not at 16 are read two tokens at a time, allowed or not."""
    rng = np.random.default_rng(V + shift)
    for density in (0.001, 0.05, 0.4, 1.0):
        allowed = rng.random((12, V)) < density
        allowed[:, -1] = True
        x = _normal(12, V, V, "bf16")
        _check(bs, x, _scores(3, 4, V), 8, allowed=allowed, uses=np.arange(12) % 4 != 1, softcap=softcap, stride=stride, shift=shift)
        same = x[:1].expand(12, V).contiguous()  # rows that begin elsewhere, but are alike: equal sums, so the lower beam goes first
        got = _check(bs, same, np.zeros((3, 4)), 8, softcap=softcap, stride=stride, shift=shift)
        assert (got["log_norms"] == got["log_norms"][0, 0]).all()
        best = int((x[0] == x[0].max()).sum())  # tokens that tie for a beam's first place; a cap of 30 leaves those behind them behind
        assert (got["parents"] == np.repeat(np.arange(4), best)[:8]).all() if best > 1 else (got["parents"][:, :4] == np.arange(4)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,stride", [(4097, 4104), (20011, 20016), (8185, 8192), (33, 40), (4097, 4097)])
def test_bits_behind_the_vocabulary_say_nothing(bs, dtype, V, stride):
    """Masks whose last word is all ones behind the last token, as compositions come out; what lies there in a row's stride is the
    largest logit of all."""
    import torch

    rng = np.random.default_rng(V)
    for dens in (0.002, 0.5):
        allowed = rng.random((6, V)) < dens
        allowed[:, V - 1] = [True, False, True, False, True, False]
        words = _words(allowed).view(np.uint32)
        words[:, -1] |= np.uint32(0xFFFFFFFF ^ ((1 << (V % 32)) - 1))
        x = _normal(6, V, 8, dtype)
        buf = torch.full((6, stride), 50.0, dtype=x.dtype, device="cuda")
        buf[:, :V] = x.cuda()
        s = _scores(2, 3, 8)
        got = bs.beam_select(buf[:, :V], torch.from_numpy(s).cuda(), 9, mask=torch.from_numpy(words.view(np.int32)).cuda(), want_norms=True)
        want, norms = beam_oracle.select(np.where(allowed, x.float().numpy(), -np.inf), s, 9)
        for b in range(2):
            n = len(want[b])
            assert [(int(p), int(t)) for p, t in zip(got["parents"][b][:n], got["tokens"][b][:n])] == [(k, v) for _, k, v, _ in want[b]]
        on = np.isfinite(norms)
        assert np.allclose(got["log_norms"].cpu().numpy()[on], norms[on], rtol=2.0 ** -24, atol=LSE)


def test_masks_of_one_word_by_any_stride(bs):
    """A dimension of one element has no stride to speak of."""
    import torch

    x, s = _normal(6, 29, 3).cuda(), torch.from_numpy(_scores(2, 3, 3)).cuda()
    words = torch.from_numpy(_words(np.random.default_rng(1).random((6, 29)) < 0.4)).cuda()
    want = bs.beam_select(x, s, 5, mask=words)
    for m in (words.t().contiguous().t(), torch.as_strided(words.flatten(), (6, 1), (1, 6)), torch.stack([words, words], 1)[:, 0]):
        got = bs.beam_select(x, s, 5, mask=m)
        assert all(torch.equal(got[k], want[k]) for k in want)


def test_mask_compose_feeds_the_selection():
    import torch

    V = 10007
    b = _sampler(max_cached_masks=4, max_vocab=V)
    try:
        rng = np.random.default_rng(1)
        sets = rng.random((2, V)) < 0.05
        for i in range(2):
            b.mask_cache_put(i + 1, _words(sets[i:i + 1])[0].view(np.uint32), V)
        keys = np.array([[1, 0], [2, 0], [1, 2], [0, 0]], np.uint64)
        mask, uses = b.mask_compose(keys, V)
        x, s = _normal(4, V, 1), _scores(1, 4, 1)
        got = b.beam_select(x.cuda(), torch.from_numpy(s).cuda(), 8, mask=mask, row_uses_mask=uses)
        on = np.stack([sets[0], sets[1], sets[0] & sets[1], np.ones(V, bool)])
        want, _ = beam_oracle.select(np.where(on, x.numpy(), -np.inf), s, 8)
        assert [(int(p), int(t)) for p, t in zip(got["parents"][0], got["tokens"][0])] == [(k, v) for _, k, v, _ in want[0]]
    finally:
        b.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_softcap_reads_as_the_capped_logits(bs, dtype):
    x = _normal(6, 20011, 3, dtype, scale=12.0)
    x[0, 3], x[1, 4] = float("inf"), float("-inf")
    _check(bs, x, _scores(2, 3, 4), 7, softcap=30.0)
    _check(bs, _normal(6, 4096, 3, dtype, scale=200.0), _scores(2, 3, 4), 7, softcap=5.0)  # most of the row at the cap


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [4097, 65536])
@pytest.mark.parametrize("garbage", [None, float("nan"), float("-inf")])
def test_softcap_behind_masks(bs, dtype, V, garbage):
    """A masked token is no candidate whatever the cap would make of it; an allowed -infinity is one at the cap's lower end."""
    rng = np.random.default_rng(V)
    allowed = rng.random((8, V)) < np.array([[0.001], [0.01], [0.05], [0.1], [0.2], [0.5], [1.0], [0.0]])
    x = _normal(8, V, 3, dtype, scale=12.0)
    x[2, 5] = x[5, 7] = float("-inf")
    allowed[2, 5] = allowed[5, 7] = True
    _check(bs, x, _scores(2, 4, 4), 9, allowed=allowed, garbage=garbage, softcap=20.0)
    _check(bs, x, _scores(4, 2, 4), 9, allowed=allowed, uses=[1, 1, 0, 1, 0, 1, 1, 0], softcap=20.0)


def test_equal_beams_go_to_the_lower_one(bs):
    """Beams that are alike in every bit: their candidates tie exactly."""
    for V, stride in ((5003, 5003), (8192, 8192), (20011, 20012)):
        x = _normal(1, V, 1).repeat(4, 1)
        got = _check(bs, x, np.full((1, 4), -1.5), 12, stride=stride)
        best = np.argsort(-x[0].numpy(), kind="stable")[:3]
        assert got["parents"][0].tolist() == [0, 1, 2, 3] * 3
        assert got["tokens"][0].tolist() == np.repeat(best, 4).tolist()


def test_many_rows():
    b = _sampler(max_rows=512, max_vocab=33000)
    try:
        _check(b, _normal(512, 3001, 8), _scores(128, 4, 8), 8)
        _check(b, _normal(400, 33000, 8, "bf16"), _scores(50, 8, 8), 16)
        _check(b, _normal(512, 500, 8), _scores(16, 32, 8), 64)
    finally:
        b.close()


def test_one_beam_is_the_arg_max(bs):
    import torch

    x = _normal(16, 50257, 3).cuda()
    idx, _ = bs.argmax_rows(x)
    got = bs.beam_select(x, torch.zeros((16, 1), device="cuda"), 1)
    assert torch.equal(got["tokens"][:, 0], idx) and (got["parents"] == 0).all()


def test_repeated_calls_and_out(bs):
    """The same call gives the same bits, into the same tensors, and different calls do not see one another."""
    import torch

    x, s = _normal(32, 30011, 3).cuda(), torch.from_numpy(_scores(8, 4, 3)).cuda()
    y, t = _normal(10, 4099, 4).cuda(), torch.from_numpy(_scores(2, 5, 3)).cuda()
    first = bs.beam_select(x, s, 8, want_norms=True)
    kept = {k: v.clone() for k, v in first.items()}
    for _ in range(20):
        bs.beam_select(y, t, 11)
        for v in first.values():
            v.fill_(-7)
        again = bs.beam_select(x, s, 8, want_norms=True, out=first)
        assert again is first
        for k in kept:
            assert torch.equal(first[k], kept[k])


def test_streams(bs):
    """Calls on different streams share the handle's workspace and are put one behind the other."""
    import torch

    x, s = [_normal(16, 60011, i).cuda() for i in range(4)], torch.from_numpy(_scores(4, 4, 3)).cuda()
    want = [bs.beam_select(v, s, 8) for v in x]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = [bs.beam_select(v, s, 8, stream=st) for v, st in zip(x, streams)]
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(g[k], w[k]) for k in w)


def test_captured_calls_have_workspace_of_their_own(bs):
    """Two graphs of one handle, replayed beside one another and beside direct calls, with new contents."""
    import torch

    s = torch.from_numpy(_scores(4, 4, 3)).cuda()
    xs = [_normal(16, 60011, i).cuda() for i in range(2)]
    outs = [bs.beam_select(x, s, 8) for x in xs]
    graphs = []
    for x, o in zip(xs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            bs.beam_select(x, s, 8, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    z = _normal(16, 60011, 77).cuda()
    for r in range(5):
        for i, x in enumerate(xs):
            x.copy_(_normal(16, 60011, 10 + 2 * r + i))
        want = [{k: v.clone() for k, v in bs.beam_select(x, s, 8).items()} for x in xs]
        torch.cuda.synchronize()
        for o in outs:
            o["tokens"].fill_(-9)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            bs.beam_select(z, s, 8)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(o[k], w[k]) for k in w)


def test_normalisers_are_closer_than_their_bound(bs):
    """Rows whose best logit is 0, beams whose score is the row's normaliser as a float: the best candidate's score is what that
    rounds off, a number so small that 32 bits show how exact the normaliser is.  The terms' errors go either way and their
    sum's is that of their mean square: with p_i the probabilities, 2^-22 * sqrt(sum p_i^2) from the exponentials and as much from
    the additions in 32 bits, five times that as a bound for the worst of 64 rows."""
    import torch

    for V, scale in ((50257, 2.5), (151936, 3.0)):
        x = _normal(64, V, 5, scale=scale)
        x[::2, :16] += 8.0  # peaked rows
        x = (x - x.amax(1, keepdim=True)).cuda()
        norm = torch.logsumexp(x.double(), 1)
        p = torch.exp(x.double() - norm[:, None])
        bound = 5 * 2 * 2.0 ** -22 * p.square().sum(1).sqrt()
        got = bs.beam_select(x, norm.float().view(64, 1), 1)
        assert ((got["scores"].view(64).double() - (norm.float().double() - norm)).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_logit_far_above_a_flat_rest(bs, dtype):
    """Rows like a model that is sure: the best logit is 0, the others lie around -17 to -20.  Beams score what the row's normaliser
    is as a float, so the best candidate's score shows the normaliser's error.  The largest term has no error of its own, and the
    rest - q of the sum - is off by no more than LSE of itself, as long as the large term takes nothing away from the small ones that
    are added up beside it (which would be up to 16 * 2^-24 of the sum).  In 64 bits the logarithm, the score and what is
    compared are off by less than 1e-14 of numbers below 32."""
    import torch

    for V, peak, scale in ((262144, 17.0, 0.5), (262144, 18.0, 1.0), (151936, 17.0, 1.0), (151936, 18.0, 0.5), (262144, 19.0, 1.5), (50257, 17.5, 1.0),
                           (50257, 20.0, 2.5)):
        x = _normal(64, V, 3, scale=scale) - peak
        at = torch.randint(0, V, (64,), generator=torch.Generator().manual_seed(V))
        x[torch.arange(64), at] = 0.0
        x = x.to(torch.bfloat16).cuda() if dtype == "bf16" else x.cuda()
        d = x.double()
        norm = torch.logsumexp(d, 1)
        q = 1.0 - torch.exp(-norm)
        got = bs.beam_select(x, norm.float().view(64, 1), 1)
        assert torch.equal(got["tokens"].view(64).cpu(), at.int())
        off = (got["scores"].view(64).double() - (norm.float().double() - norm)).abs()
        assert (off <= q * LSE + 1e-12 + 2.0 ** -24 * (norm.float().double() - norm).abs()).all(), (V, peak, scale, float((off / (q * LSE)).max()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("peak", [16.75, 17.0, 17.375, 18.0])
def test_large_logits_do_not_swallow_the_small_ones_beside_them(bs, dtype, peak):
    """One logit of 0 in every thread's share of a group, n elements, the others at -peak, of which one alone is less than half a
    step of the sum.  The terms of a share are added pair by pair, so a large one takes part in log2(n) additions, each rounded by
    2^-24 of it; the others' own errors are of no account, as all of them together are less than 1e-6 of the sum.  (Added
    one after the other, each would be lost: n / 2 * e^-peak of the sum.)"""
    import torch

    V, n = 131072, 32 if dtype == "bf16" else 16
    x = torch.full((8, V // (32 * n), 32 * n), -peak)
    x[:, :, :8 * n:n // 4] = 0.0  # a thread reads n / 4 neighbours at a time
    x = x.view(8, V).to(torch.bfloat16 if dtype == "bf16" else torch.float32).cuda()
    norm = torch.logsumexp(x.double(), 1)
    got = bs.beam_select(x, norm.float().view(8, 1), 1)
    exact = norm.float().double() - norm  # the best candidate's score
    off = (got["scores"].view(8).double() - exact).abs()
    assert (got["tokens"] == 0).all()
    assert (off <= np.log2(n) * 2.0 ** -24 + 1e-9 + 2.0 ** -24 * exact.abs()).all(), float(off.max())


def test_more_rows_than_a_grid_has_in_one_dimension():
    import torch

    b = _sampler(max_rows=66000, max_vocab=64, max_history=1, max_top_k=1)
    try:
        x = torch.randn((66000, 40), generator=torch.Generator().manual_seed(2)).cuda()
        got = b.beam_select(x, torch.zeros((66000, 1), device="cuda"), 2)
        best = x.topk(2, 1)
        assert torch.equal(got["tokens"].long(), best.indices)
        lp = best.values.double() - torch.logsumexp(x.double(), 1, keepdim=True)
        assert ((got["scores"] - lp).abs() <= 2 * LSE + lp.abs() * 2.0 ** -24).all()
    finally:
        b.close()


def test_outputs_stay_within_their_tensors(bs):
    import torch

    x, s = _normal(12, 3001, 2).cuda(), torch.from_numpy(_scores(3, 4, 2)).cuda()
    wide = {k: torch.full((5, 9), -77, dtype=d, device="cuda") for k, d in (("tokens", torch.int32), ("parents", torch.int32), ("scores", torch.float32))}
    out = bs.beam_select(x, s, 9, out={k: v[1:4] for k, v in wide.items()})
    want = bs.beam_select(x, s, 9)
    for k, v in wide.items():
        assert torch.equal(out[k], want[k]) and (v[0] == -77).all() and (v[4] == -77).all()


def test_refusals(bs):
    import torch
    from opentail.stingray_b200 import StingrayError

    x, s = torch.zeros((8, 100), device="cuda"), torch.zeros((2, 4), device="cuda")
    with pytest.raises(StingrayError, match="128"):
        bs.beam_select(x, s, 129)
    with pytest.raises(StingrayError):
        bs.beam_select(x, s, 0)
    with pytest.raises(StingrayError, match="32"):
        bs.beam_select(torch.zeros((33, 100), device="cuda"), torch.zeros((1, 33), device="cuda"), 4)
    with pytest.raises(StingrayError, match="max_rows"):
        bs.beam_select(torch.zeros((68, 100), device="cuda"), torch.zeros((17, 4), device="cuda"), 4)
    with pytest.raises(StingrayError, match="max_vocab"):
        bs.beam_select(torch.zeros((1, 262145), device="cuda"), torch.zeros((1, 1), device="cuda"), 4)
    with pytest.raises(StingrayError, match="softcap"):
        bs.beam_select(x, s, 4, softcap=-1.0)
    for bad in (x.half(), x[:7], x.cpu(), x.t().contiguous().t()):
        with pytest.raises(ValueError):
            bs.beam_select(bad, s, 4)
    for bad in (s.double(), s.cpu(), s.t().contiguous().t()):
        with pytest.raises(ValueError):
            bs.beam_select(x, bad, 4)
    with pytest.raises(ValueError):
        bs.beam_select(x, s, 4, mask=torch.zeros((8, 3), dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        bs.beam_select(x, s, 4, row_uses_mask=torch.zeros(8, dtype=torch.uint8, device="cuda"))
    out = bs.beam_select(x, s, 4)
    with pytest.raises(ValueError):
        bs.beam_select(x, s, 5, out=out)
    empty = bs.beam_select(torch.zeros((0, 100), device="cuda"), torch.zeros((0, 4), device="cuda"), 4)
    assert empty["tokens"].shape == (0, 4)


def test_guards_hold():
    import torch
    from tests.test_gpu_checked_handle import _checked, _guards

    b = _checked(max_rows=33, max_vocab=20011, max_history=8, max_top_k=8)
    try:
        for K, n in ((32, 128), (1, 128), (11, 5)):
            B = 33 // K
            for V in (20011, 20000, 40):
                b.beam_select(_normal(B * K, V, 1).cuda(), torch.from_numpy(_scores(B, K, 1)).cuda(), n)
        count, bad = _guards(b)
        assert count > 20 and bad == -1
    finally:
        b.close()
