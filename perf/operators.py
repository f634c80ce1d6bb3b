"""Beam search over the library's rows, as cases that can be timed and compared.

A program that decodes with beams keeps ``num_beams`` rows of logits per sequence and does four things per
token or per request.  Kinds (``case["kind"]``):

  select   ``BatchSampler.beam_select``: the best continuations of every sequence over its beams and the
           vocabulary - log-softmax of each row, the beams' running scores, the ``n`` best of beams x vocabulary -
           and each row's normaliser, from which a program takes the log-probability of any other token
  steps    ``BatchSampler.beam_start`` and a few ``beam_advance``: candidates into continuing beams, ended
           hypotheses into the sequence's pool of best ones; then the pool's sequences out of the trail
  reorder  ``BatchSampler.beam_reorder``: per-beam state (key/value caches up to the positions in use, recurrent
           states, page tables) follows the beams that continue, in place
  trace    ``BatchSampler.beam_backtrace``: the token sequences of hypotheses out of the trail

Scores are compared in 64 bits: two beams' candidates can lie closer together than 32 bits tell apart.  Equal
scores go to the lower beam, and within a beam to the larger logit, then to the lower token.
"""
import math

import torch

own = False

SHORT, LONG = 32_000, 262_144  # vocabularies of the tests and configurations lie between these
MAX_ROWS = 512
EOS, PAD = 2, 0


# ---- the cases -----------------------------------------------------------------------------------------

def _select(name, n_seq, beams, vocab, dtype="f32", n=0, mask=False, first=False, logits="peaked"):
    c = {"kind": "select", "n_seq": n_seq, "beams": beams, "vocab": vocab, "dtype": dtype, "n": n or 2 * beams, "mask": mask, "first": first,
         "logits": logits}
    return dict(c, name=name) if name else c


def _steps(name, n_seq, beams, steps, room, n=0):
    c = {"kind": "steps", "n_seq": n_seq, "beams": beams, "steps": steps, "room": room, "n": n or 2 * beams}
    return dict(c, name=name) if name else c


def _reorder(name, n_seq, beams, layout, dtype, tensors, heads, room, width, ragged=False):
    c = {"kind": "reorder", "n_seq": n_seq, "beams": beams, "layout": layout, "dtype": dtype, "tensors": tensors, "heads": heads, "room": room,
         "width": width, "ragged": ragged}
    return dict(c, name=name) if name else c


def _trace(name, n_seq, beams, steps):
    c = {"kind": "trace", "n_seq": n_seq, "beams": beams, "steps": steps}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one request with four beams on the single-row configuration's vocabulary: latency
        _select("select_chat", 1, 4, 151_936),
        # a few requests on an odd vocabulary, rows not aligned, a wider choice than two per beam
        _select("select_ragged", 6, 5, 50_257, n=13),
        # a server's step: 256 rows of the headline configuration as 64 requests of four beams
        _select("select_server", 64, 4, 151_936, logits="flat"),
        # structured output with beams: a bitmask of allowed tokens per row (the grammar configuration)
        _select("select_grammar", 16, 4, 262_144, dtype="bf16", mask=True, logits="flat"),
        # wide beams, one GPU's rows of the large configuration with bf16 logits
        _select("select_wide", 32, 16, 256_000, dtype="bf16"),
        # one request of sixteen tokens behind the selection, to its end
        _steps("steps_chat", 1, 4, 16, 16),
        # a few tokens of a full server, with room for more
        _steps("steps_server", 64, 8, 4, 64),
        # the key/value caches of eight layers of one request, 1000 of 1024 positions in use
        _reorder("reorder_chat", 1, 4, "kv", "bf16", 16, 8, 1024, 128),
        # recurrent states of a small model, odd sizes, fp32
        _reorder("reorder_states", 7, 5, "state", "f32", 6, 16, 63, 33),
        # the caches of four layers of a server, every request at a position of its own
        _reorder("reorder_server", 32, 8, "kv", "bf16", 8, 8, 768, 128, ragged=True),
        # a short answer's hypotheses
        _trace("trace_chat", 1, 4, 256),
        # a server's long answers
        _trace("trace_server", 64, 8, 4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))


def draw(rng):
    """Another case of the same ranges.  Vocabularies from 32,000 to 262,144, mostly padded to a multiple of 64 as
    model heads are, some only even or odd; 1 to 32 beams; no case costs more than the largest listed one."""
    kind = rng.choice(["select", "select", "select", "steps", "reorder", "reorder", "trace"])
    beams = rng.choice([2, 3, 4, 4, 5, 8, _log_int(rng, 1, 32)])
    if kind == "select":
        vocab, pad = _log_int(rng, SHORT, LONG), rng.choice([64, 64, 64, 8, 2, 1])
        vocab = min(LONG, (vocab + pad - 1) // pad * pad)
        n_seq = max(1, min(_log_int(rng, 1, MAX_ROWS // beams), 60_000_000 // (vocab * beams)))
        n = rng.choice([2 * beams, 2 * beams, beams, 3 * beams, 2 * beams + 1])
        return _select(None, n_seq, beams, vocab, rng.choice(["f32", "bf16"]), min(n, 128), rng.random() < 0.25, rng.random() < 0.15,
                       rng.choice(["flat", "peaked"]))
    if kind == "steps":
        steps = _log_int(rng, 1, 16)
        return _steps(None, _log_int(rng, 1, MAX_ROWS // beams), beams, steps, steps + rng.choice([0, 0, 1, 50]), rng.choice([beams, 2 * beams, 3 * beams]))
    if kind == "reorder":
        n_seq = _log_int(rng, 1, max(1, 256 // beams))
        layout, dtype = rng.choice(["kv", "kv", "kv", "kv_last", "state", "pages"]), rng.choice(["bf16", "bf16", "f32"])
        heads, width = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 80, 33])
        room = _log_int(rng, 16, 2048)
        one = n_seq * beams * heads * width * room * (4 if dtype == "f32" else 2)
        tensors = max(1, min(rng.choice([1, 2, 8, 16]), 400_000_000 // one))
        room = max(1, min(room, room * 400_000_000 // one))
        return _reorder(None, n_seq, beams, layout, dtype, tensors, heads, room, width, rng.random() < 0.5)
    n_seq = _log_int(rng, 1, max(1, MAX_ROWS // beams))
    return _trace(None, n_seq, beams, max(1, min(_log_int(rng, 1, 4096), 2_000_000 // (n_seq * beams))))


# ---- inputs --------------------------------------------------------------------------------------------

def _logits(g, rows, vocab, how, dtype, dev):
    """flat: N(0, 2.5^2), as in the configurations.  peaked: N(0, 3^2) with 16 ids boosted by 2 to 10, the
    shape a model's head gives when it has an idea what comes next."""
    x = torch.randn((rows, vocab), generator=g, device=dev)
    x *= 2.5 if how == "flat" else 3.0
    if how == "peaked":
        ids = torch.randint(0, vocab, (rows, 16), generator=g, device=dev)
        x.scatter_add_(1, ids, 2.0 + 8.0 * torch.rand((rows, 16), generator=g, device=dev))
    return x.to(torch.bfloat16) if dtype == "bf16" else x


def _mask(g, rows, vocab, dev):
    """Allowed-token bits, density log-uniform in [0.1 %, 30 %], at least one bit set per row."""
    words = (vocab + 31) // 32
    dens = torch.exp(torch.empty(rows, 1, device=dev).uniform_(math.log(0.001), math.log(0.30), generator=g))
    bits = torch.zeros((rows, words * 32), dtype=torch.bool, device=dev)
    bits[:, :vocab] = torch.rand((rows, vocab), generator=g, device=dev) < dens
    bits[torch.arange(rows, device=dev), torch.randint(0, vocab, (rows,), generator=g, device=dev)] = True
    weights = torch.ones(32, dtype=torch.int64, device=dev) << torch.arange(32, device=dev)
    out = torch.empty((rows, words), dtype=torch.int32, device=dev)
    for r in range(0, rows, 32):  # a block of rows at a time: the sum below is 64-bit
        v = (bits[r:r + 32].view(-1, words, 32).to(torch.int64) * weights).sum(-1)
        out[r:r + 32] = torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)
    return out


def _parents(g, shape, beams, dev):
    """Which beam each beam continues: some end, some continue more than once."""
    weight = torch.rand(shape[:-1] + (beams,), generator=g, device=dev).square().add_(0.01)
    return torch.multinomial(weight.view(-1, beams), shape[-1], replacement=True, generator=g).view(shape).to(torch.int32)


class _State:
    pass


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    s = _State()
    s.kind, s.n_seq, s.beams = case["kind"], case["n_seq"], case["beams"]
    s.dev, s.kept = dev, None
    B, K = s.n_seq, s.beams
    if s.kind == "select":
        s.n = case["n"]
        s.logits = _logits(g, B * K, case["vocab"], case["logits"], case["dtype"], dev)
        s.mask = _mask(g, B * K, case["vocab"], dev) if case["mask"] else None
        s.scores = -torch.rand((B, K), generator=g, device=dev).mul_(4.0).cumsum(1)
        if case["first"]:  # a request's first token: one beam that is alive
            s.scores[:, 0] = 0.0
            s.scores[:, 1:] = -math.inf
    elif s.kind == "steps":
        s.n, s.steps, s.room = case["n"], case["steps"], case["room"]
        S, n = s.steps, s.n
        s.tokens = torch.randint(3, SHORT, (S, B, n), generator=g, device=dev, dtype=torch.int32)
        s.tokens[torch.rand((S, B, n), generator=g, device=dev) < 0.15] = EOS
        s.parents = torch.randint(0, K, (S, B, n), generator=g, device=dev, dtype=torch.int32)
        start = torch.arange(S, device=dev).view(S, 1, 1) * 1.5 + 0.1
        s.scores = -(start + torch.rand((S, B, n), generator=g, device=dev).mul_(0.8).cumsum(2))
    elif s.kind == "reorder":
        s.layout, s.ragged, room = case["layout"], case["ragged"], case["room"]
        R, H, D = B * K, case["heads"], case["width"]
        shape = {"kv": (R, H, room, D), "kv_last": (R, H, D, room), "state": (R, H, room * D), "pages": (R, room)}[s.layout]
        if s.layout == "pages":
            s.tensors = [torch.randint(0, 1 << 30, shape, generator=g, device=dev, dtype=torch.int32) for _ in range(case["tensors"])]
        else:
            dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
            s.tensors = [torch.randn(shape, generator=g, device=dev).to(dtype) for _ in range(case["tensors"])]
        s.parents = _parents(g, (B, K), K, dev)
        s.position_dim = {"kv": 2, "kv_last": 3, "state": None, "pages": 1}[s.layout]
        s.positions = None
        if s.position_dim is not None:
            used = max(1, room * 125 // 128)
            s.positions = torch.randint(max(1, used // 2), used + 1, (B,), generator=g, device=dev, dtype=torch.int32) if s.ragged else used
    else:
        s.steps = case["steps"]
        s.tokens = torch.randint(3, SHORT, (s.steps, B, K), generator=g, device=dev, dtype=torch.int32)
        s.parents = _parents(g, (s.steps, B, K), K, dev)
        low = s.steps // 2
        s.ends = torch.randint(low, s.steps, (B, K), generator=g, device=dev, dtype=torch.int32)
        s.end_parents = torch.randint(0, K, (B, K), generator=g, device=dev, dtype=torch.int32)
        s.end_tokens = torch.full((B, K), EOS, device=dev, dtype=torch.int32)
    return s


# ---- the plain form ------------------------------------------------------------------------------------

def _allowed(mask, vocab):
    bit = torch.arange(32, device=mask.device, dtype=torch.int32)
    return ((mask.unsqueeze(-1) >> bit) & 1).bool().flatten(1)[:, :vocab]


def _plain_select(s):
    rows, vocab = s.logits.shape
    B, K, n = s.n_seq, s.beams, s.n
    x = s.logits.float()
    if s.mask is not None:
        x = x.masked_fill(~_allowed(s.mask, vocab), -math.inf)
    top = x.amax(1, keepdim=True).double()
    norm = (x.double() - top).exp_().sum(1, keepdim=True).log_() + top
    # the n best of a row: by logit, equal ones by token, as one whole number per element
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + ((1 << 32) - 1 - torch.arange(vocab, device=s.dev))
    key = key.topk(min(n, vocab), dim=1).values
    token = (1 << 32) - 1 - (key & 0xFFFFFFFF)
    score = x.gather(1, token).double() - norm + s.scores.view(rows, 1).double()
    score = score.masked_fill((s.scores.view(rows, 1) == -math.inf) | (x.gather(1, token) == -math.inf), -math.inf)
    score, token = score.view(B, -1), token.view(B, -1)
    beam = torch.arange(K, device=s.dev).repeat_interleave(score.shape[1] // K).expand(B, -1)
    score, order = score.sort(dim=1, descending=True, stable=True)
    score, order = score[:, :n], order[:, :n]
    none = score == -math.inf
    return {"tokens": token.gather(1, order).masked_fill(none, -1).int(), "parents": beam.gather(1, order).masked_fill(none, -1).int(),
            "scores": score.float(), "log_norms": torch.where(s.scores == -math.inf, -math.inf, norm.view(B, K)).float()}


def _plain_steps(s):
    B, K, S, T, n, dev = s.n_seq, s.beams, s.steps, s.room, s.n, s.dev
    low = -math.inf
    slot = torch.arange(K, device=dev, dtype=torch.int32).expand(B, K)
    done = torch.zeros(B, dtype=torch.bool, device=dev)
    count = torch.zeros(B, dtype=torch.int32, device=dev)
    pool = [torch.full((B, K), low, device=dev)] + [torch.full((B, K), -1, dtype=torch.int32, device=dev) for _ in range(3)]
    trail = [torch.full((T, B, K), PAD, dtype=torch.int32, device=dev), slot.expand(T, B, K).clone()]
    for t in range(S):
        tok, par, sc = s.tokens[t], s.parents[t], s.scores[t]
        on = ~done
        end = tok == EOS
        place = (~end).long().cumsum(1) - 1
        place = torch.where(~end & (place < K), place, K)  # the others go behind the last beam
        nt = torch.full((B, K + 1), PAD, dtype=torch.int32, device=dev).scatter(1, place, tok)[:, :K]
        np_ = torch.cat([slot, slot[:, :1]], 1).scatter(1, place, par)[:, :K]
        ns = torch.full((B, K + 1), low, device=dev).scatter(1, place, sc)[:, :K]
        norm = float(t + 1)
        hit = end & (torch.arange(n, device=dev) < K) & on[:, None]
        new = [torch.where(hit, (sc.double() / norm).float(), low), torch.where(hit, t, -1).int(), torch.where(hit, par, -1), torch.where(hit, tok, -1)]
        if t + 1 == T:  # the last step there is room for: what continues is a hypothesis too
            alive = (ns > low) & on[:, None]
            last = [torch.where(alive, (ns.double() / norm).float(), low), torch.where(alive, t, -1).int(), torch.where(alive, np_, -1),
                    torch.where(alive, nt, -1)]
            new = [torch.cat(v, 1) for v in zip(new, last)]
        every = [torch.cat(v, 1) for v in zip(pool, new)]
        order = every[0].sort(dim=1, descending=True, stable=True).indices[:, :K]
        pool = [v.gather(1, order) for v in every]
        trail[0][t], trail[1][t] = nt, np_
        count = count + on.int()
        over = (ns[:, 0] == low) | ((pool[0][:, -1] > low) & (pool[0][:, -1] >= (ns[:, 0].double() / norm).float()))
        done = done | over if t + 1 < T else torch.ones_like(done)
    return {"tokens": torch.where(done[:, None], PAD, nt).int(), "parents": torch.where(done[:, None], slot, np_), "scores": torch.where(done[:, None], low, ns),
            "steps": count, "done": done.int(), "pool_scores": pool[0], "pool_steps": pool[1], "pool_parents": pool[2], "pool_tokens": pool[3],
            **_sequences(*trail, *pool[1:])}


def _plain_reorder(s):
    K = s.beams
    source = (torch.arange(s.n_seq, device=s.dev)[:, None] * K + s.parents).flatten()
    for t in s.tensors:
        moved = t.index_select(0, source)
        if s.positions is None:
            t.copy_(moved)
        elif s.ragged:
            at = torch.arange(t.shape[s.position_dim], device=s.dev).view([-1 if d == s.position_dim else 1 for d in range(t.dim())])
            used = s.positions.repeat_interleave(K).view([-1] + [1] * (t.dim() - 1))
            t.copy_(torch.where(at < used, moved, t))
        else:
            t.narrow(s.position_dim, 0, s.positions).copy_(moved.narrow(s.position_dim, 0, s.positions))
    return s.tensors


def _sequences(tokens, parents, ends, end_parents, end_tokens):
    T = tokens.shape[0]
    out = torch.full((T,) + ends.shape, PAD, dtype=torch.int32, device=ends.device)
    beam = end_parents.clamp(min=0).long()
    for t in range(T - 1, -1, -1):
        at, before = ends == t, ends > t
        out[t] = torch.where(before, tokens[t].gather(1, beam), torch.where(at, end_tokens, PAD))
        beam = torch.where(before, parents[t].gather(1, beam).long(), beam)
    return {"sequences": out.permute(1, 2, 0).contiguous(), "lengths": ends + 1}


def _plain_trace(s):
    return _sequences(s.tokens, s.parents, s.ends, s.end_parents, s.end_tokens)


# ---- the framework's operators -------------------------------------------------------------------------

_handle = None


def _sampler():
    """The program's one library handle, as wide as the largest case."""
    global _handle
    if _handle is None:
        from opentail.stingray_b200 import BatchSampler

        _handle = BatchSampler(max_rows=MAX_ROWS, max_vocab=LONG, max_history=1, max_top_k=1)
    return _handle


def _own(s):
    b = _sampler()
    if s.kind == "select":
        s.kept = b.beam_select(s.logits, s.scores, s.n, mask=s.mask, want_norms=True, out=s.kept)
        return s.kept
    if s.kind == "steps":
        if s.kept is None:
            from opentail.stingray_b200 import BeamSearch

            s.kept = BeamSearch(s.n_seq, s.beams, s.room, eos=[EOS], pad=PAD, length_penalty=1.0, device=s.dev)
            s.found = None
        k = s.kept
        b.beam_start(k)
        for t in range(s.steps):
            b.beam_advance(k, {"tokens": s.tokens[t], "parents": s.parents[t], "scores": s.scores[t]})
        s.found = b.beam_backtrace(k.trail_tokens, k.trail_parents, k.pool_steps, k.pool_parents, k.pool_tokens, pad=PAD, out=s.found)
        return {"tokens": k.tokens, "parents": k.parents, "scores": k.scores, "steps": k.steps, "done": k.done, "pool_scores": k.pool_scores,
                "pool_steps": k.pool_steps, "pool_parents": k.pool_parents, "pool_tokens": k.pool_tokens, **s.found}
    if s.kind == "reorder":
        if s.kept is None:
            from opentail.stingray_b200 import BeamStates

            s.kept = BeamStates(s.tensors, s.beams, position_dim=s.position_dim)
        b.beam_reorder(s.kept, s.parents, positions=s.positions)
        return s.tensors
    s.kept = b.beam_backtrace(s.tokens, s.parents, s.ends, s.end_parents, s.end_tokens, pad=PAD, out=s.kept)
    return s.kept


def run(s):
    if own:
        return _own(s)
    return {"select": _plain_select, "steps": _plain_steps, "reorder": _plain_reorder, "trace": _plain_trace}[s.kind](s)


# ---- what a pass cannot do without, and what it returns in 64 bits ---------------------------------------

def _read_share(per_sector):
    """The share of a row's 32-byte sectors that hold an allowed token, for densities log-uniform in [0.1 %, 30 %]."""
    steps = 200
    at = [math.exp(math.log(0.001) + (math.log(0.30) - math.log(0.001)) * (i + 0.5) / steps) for i in range(steps)]
    return sum(1.0 - (1.0 - d) ** per_sector for d in at) / steps


def work(case):
    B, K = case["n_seq"], case["beams"]
    if case["kind"] == "select":
        esz = 2 if case["dtype"] == "bf16" else 4
        rows, vocab = B if case["first"] else B * K, case["vocab"]
        share = _read_share(32 // esz) if case["mask"] else 1.0
        read = rows * vocab * esz * share + (rows * ((vocab + 31) // 32) * 4 if case["mask"] else 0)
        return {"bytes": read + B * K * 4 + B * case["n"] * 12, "flops": 4 * rows * vocab * share}
    if case["kind"] == "steps":
        return {"bytes": case["steps"] * B * (case["n"] * 12 + K * 8) + B * K * (36 + 4 * case["room"]), "flops": case["steps"] * B * case["n"]}
    if case["kind"] == "reorder":
        each = {"bf16": 2, "f32": 4}[case["dtype"]]
        used = max(1, case["room"] * 125 // 128)
        used = 0.75 * used if case["ragged"] and case["layout"] != "state" else case["room"] if case["layout"] == "state" else used
        row = used * 4 if case["layout"] == "pages" else case["heads"] * used * case["width"] * each
        # of K beams that continue beams drawn with squared uniform weights about 0.55 K different ones are read, and
        # all but about one are written elsewhere than they came from
        return {"bytes": case["tensors"] * B * row * (max(1.0, 0.55 * K) + (K - 1)), "flops": 0}
    T = case["steps"]
    return {"bytes": T * B * K * (4 + 4 * 0.75 + 4), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "select":
        rows, vocab = s.logits.shape
        parts, norms = [], []
        for b in range(s.n_seq):  # a sequence at a time
            x = s.logits[b * s.beams:(b + 1) * s.beams].double()
            if s.mask is not None:
                x[~_allowed(s.mask[b * s.beams:(b + 1) * s.beams], vocab)] = -math.inf
            norms.append(torch.logsumexp(x, 1).masked_fill(s.scores[b] == -math.inf, -math.inf))
            x = x - torch.logsumexp(x, 1, keepdim=True) + s.scores[b].double()[:, None]
            parts.append(x.flatten().topk(s.n).values)
        return {"tokens": None, "parents": None, "scores": torch.stack(parts), "log_norms": torch.stack(norms)}
    if s.kind == "steps":
        tok, sc = s.tokens.cpu().tolist(), s.scores.double().cpu().tolist()
        pools, lives = [], []
        for b in range(s.n_seq):
            pool, kept, over = [], [], False
            for t in range(s.steps):
                if over:
                    break
                kept = [v for v, k in zip(sc[t][b], tok[t][b]) if k != EOS][:s.beams]
                ended = [v / (t + 1) for i, (v, k) in enumerate(zip(sc[t][b], tok[t][b])) if k == EOS and i < s.beams]
                if t + 1 == s.room:
                    ended += [v / (t + 1) for v in kept]
                pool = sorted(pool + ended, reverse=True)[:s.beams]
                over = t + 1 == s.room or not kept or (len(pool) == s.beams and pool[-1] >= kept[0] / (t + 1))
            pools.append(pool + [-math.inf] * (s.beams - len(pool)))
            kept = [] if over else kept
            lives.append(kept + [-math.inf] * (s.beams - len(kept)))
        out = dict.fromkeys(("tokens", "parents", "scores", "steps", "done", "pool_scores", "pool_steps", "pool_parents", "pool_tokens", "sequences", "lengths"))
        return out | {"scores": torch.tensor(lives, dtype=torch.float64), "pool_scores": torch.tensor(pools, dtype=torch.float64)}
    if s.kind == "reorder":
        if s.layout == "pages":
            return [None] * len(s.tensors)
        out, parents = [], s.parents.cpu().tolist()
        used = s.positions.cpu().tolist() if s.ragged and s.positions is not None else [s.positions] * s.n_seq
        for t in s.tensors:
            new = t.clone()
            for b in range(s.n_seq):
                for k in range(s.beams):
                    to, of = new[b * s.beams + k], t[b * s.beams + parents[b][k]]
                    if s.positions is not None:
                        to, of = to.narrow(s.position_dim - 1, 0, used[b]), of.narrow(s.position_dim - 1, 0, used[b])
                    to.copy_(of)
            out.append(new)
        return out
    return None
