"""The head of a language model - the product with the vocabulary - as cases that can be timed and compared.

The library's rows of logits come out of a head: hidden states ``[rows, width]`` times a weight ``[vocab, width]``.  A
program scores tokens with it, trains it, and decodes with it.  Kinds (``case["kind"]``):

  score    ``BatchSampler.head_loss``: minus the log-probability of one token per row (softmax cross entropy) and each row's
           normaliser, straight from hidden states and weight, in pieces of the vocabulary: no logits are kept
  train    ``head_loss`` and ``BatchSampler.head_loss_backward``: the same, then the gradients of the hidden states and of
           the weight for given gradients of the losses
  logits   ``BatchSampler.head_logits``: the logits of a decode step from a weight held in 4 bits with a scale (and
           a zero point) per group of columns, for the sampling calls that follow

A row whose target is below 0 has no loss: it is padding or a prompt, and its hidden state may hold anything.
"""
import math

import torch

own = False

SHORT, LONG = 32_000, 262_144  # vocabularies of the tests and configurations lie between these
MAX_ROWS = 256                 # of a decode step
PIECE = 8192                   # vocabulary entries the plain form takes at a time
MOST = 8192 * 4096 * 151_936   # rows x width x vocabulary of the largest training step


# ---- the cases -----------------------------------------------------------------------------------------

def _loss(kind, name, rows, width, vocab, dtype="bf16", ignored=0.0, softcap=0.0):
    c = {"kind": kind, "rows": rows, "width": width, "vocab": vocab, "dtype": dtype, "ignored": ignored, "softcap": softcap}
    return dict(c, name=name) if name else c


def _logits(name, rows, width, vocab, group, dtype="bf16", scales="f16", zeros=False, out="f32"):
    c = {"kind": "logits", "rows": rows, "width": width, "vocab": vocab, "group": group, "dtype": dtype, "scales": scales, "zeros": zeros, "out": out}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the last tokens of one request, scored by a small model on an odd vocabulary: latency
        _loss("score", "score_few", 5, 1024, 50_257),
        # the tokens a decode step of the single-row configuration's vocabulary came up with, scored by a large head: one reading of the weight
        _loss("score", "score_step", 64, 4096, 151_936),
        # a window of a perplexity run over the large vocabulary, with a soft cap, ragged
        _loss("score", "score_window", 1000, 2560, 262_144, dtype="f16", softcap=30.0),
        # the evaluation of a training batch
        _loss("score", "score_batch", 8192, 4096, 151_936),
        # a small tuning step in fp16, a few padded rows
        _loss("train", "train_few", 100, 1024, 32_000, dtype="f16", ignored=0.1),
        # instruction tuning: most tokens are prompts
        _loss("train", "train_tuning", 2047, 2048, 151_936, ignored=0.6),
        # pretraining
        _loss("train", "train_batch", 8192, 4096, 151_936),
        # one token of one request
        _logits("logits_token", 1, 4096, 151_936, 32),
        # a small model's odd vocabulary, a few requests, zero points
        _logits("logits_small", 3, 896, 50_257, 64, dtype="f16", zeros=True),
        # sixteen beams on the large vocabulary, bf16 logits
        _logits("logits_beams", 16, 2048, 256_000, 128, scales="bf16", out="bf16"),
        # a server's step: the headline configuration's 256 rows
        _logits("logits_server", 256, 4096, 151_936, 128, zeros=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))


def _vocab(rng):
    """Mostly padded to a multiple of 64 as model heads are, some only even or odd."""
    pad = rng.choice([64, 64, 64, 8, 2, 1])
    return min(LONG, (_log_int(rng, SHORT, LONG) + pad - 1) // pad * pad)


def draw(rng):
    """Another case of the same ranges: widths from 512 to 4096 in steps of 8 (of a group where there are groups), 1 to
    8192 rows (a decode step: to 256); no case costs more than the largest listed one."""
    kind = rng.choice(["score", "score", "train", "train", "logits", "logits", "logits"])
    vocab = _vocab(rng)
    if kind == "logits":
        group = rng.choice([32, 64, 128])
        width = max(512 // group, _log_int(rng, 512, 4096) // group) * group
        rows = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 1, MAX_ROWS), _log_int(rng, 1, MAX_ROWS)])
        return _logits(None, rows, width, vocab, group, rng.choice(["bf16", "bf16", "f16"]), rng.choice(["f16", "bf16"]), rng.random() < 0.4,
                       rng.choice(["f32", "f32", "bf16"]))
    step = rng.choice([64, 64, 8])
    width = _log_int(rng, 512, 4096) // step * step
    rows = max(1, min(_log_int(rng, 1, 8192), MOST // (width * vocab)))
    return _loss(kind, None, rows, width, vocab, rng.choice(["bf16", "bf16", "f16"]), rng.choice([0.0, 0.0, 0.1, 0.6]), rng.choice([0.0, 0.0, 30.0]))


# ---- inputs --------------------------------------------------------------------------------------------

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ignored(case):
    return int(case["rows"] * case["ignored"])


class _State:
    pass


def prepare(case, seed):
    """Hidden states of unit variance and a weight that give logits N(0, 2.5^2); a row's hidden state leans towards its
    target, by 1 to 4 units of its weight row's direction: some targets are expected, others are not."""
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    s = _State()
    s.dev, s.kind, s.kept = dev, case["kind"], None
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    dtype = _TYPES[case["dtype"]]
    if s.kind == "logits":
        s.group, s.out = case["group"], _TYPES[case["out"]]
        s.hidden = torch.randn((rows, width), generator=g, device=dev).to(dtype)
        s.codes = torch.randint(0, 256, (vocab, width // 2), generator=g, device=dev, dtype=torch.uint8)  # two columns to a byte, the lower half first
        # uniform codes about 8 (or a zero point about 7.5) have a deviation of 4.6
        s.scales = ((0.5 + torch.rand((vocab, width // s.group), generator=g, device=dev)) * (2.5 / 4.6 / math.sqrt(width))).to(_TYPES[case["scales"]])
        s.zeros = None
        if case["zeros"]:
            s.zeros = (6.0 + 3.0 * torch.rand((vocab, width // s.group), generator=g, device=dev)).to(s.scales.dtype)
        if own:  # the weight is laid out once, when the model is loaded
            s.packed = _sampler().head_pack(s.codes, s.scales, s.zeros)
        return s
    s.softcap = case["softcap"]
    s.weight = torch.empty((vocab, width), dtype=dtype, device=dev)
    for v in range(0, vocab, 16384):
        n = min(16384, vocab - v)
        s.weight[v:v + n] = torch.randn((n, width), generator=g, device=dev).mul_(2.5 / math.sqrt(width))
    s.targets = torch.randint(0, vocab, (rows,), generator=g, device=dev, dtype=torch.int32)
    lean = 1.0 + 3.0 * torch.rand((rows, 1), generator=g, device=dev)
    s.hidden = (torch.randn((rows, width), generator=g, device=dev) + lean / 2.5 * s.weight[s.targets.long()].float()).to(dtype)
    s.targets[torch.randperm(rows, generator=g, device=dev)[:_ignored(case)]] = -100
    s.grad_loss = torch.where(s.targets >= 0, 1.0 / max(1, rows - _ignored(case)), 0.0)
    if s.kind == "train":
        s.grad_loss *= 0.5 + torch.rand(rows, generator=g, device=dev)  # weights of the tokens
    return s


# ---- the plain form ------------------------------------------------------------------------------------

def _capped(s, rows, piece):
    """Logits of some rows for a piece of the vocabulary, and what the soft cap makes of their gradients."""
    x = rows @ piece.float().T
    if not s.softcap:
        return x, None
    t = torch.tanh(x / s.softcap)
    return t * s.softcap, 1.0 - t * t


def _plain_loss(s):
    used = (s.targets >= 0).nonzero().flatten()
    rows, targets = s.hidden[used].float(), s.targets[used].long()
    n, vocab = rows.shape[0], s.weight.shape[0]
    top = torch.full((n,), -math.inf, device=s.dev)
    total = torch.zeros(n, dtype=torch.float64, device=s.dev)
    hit = torch.zeros(n, device=s.dev)
    for v in range(0, vocab, PIECE):
        x, _ = _capped(s, rows, s.weight[v:v + PIECE])
        new = torch.maximum(top, x.amax(1))
        total = total * torch.exp((top - new).double()) + torch.exp(x - new[:, None]).sum(1)
        top = new
        at = targets - v
        here = (at >= 0) & (at < x.shape[1])
        hit = torch.where(here, x.gather(1, at.clamp(0, x.shape[1] - 1)[:, None])[:, 0], hit)
    norm = torch.log(total) + top.double()
    loss, norms = (torch.zeros(s.targets.shape[0], device=s.dev) for _ in range(2))
    loss[used] = (norm - hit.double()).float()
    norms[used] = norm.float()
    return {"loss": loss, "log_norms": norms}


def _plain_train(s):
    out = _plain_loss(s)
    used = (s.targets >= 0).nonzero().flatten()
    rows, targets = s.hidden[used].float(), s.targets[used].long()
    norms, scale = out["log_norms"][used], s.grad_loss[used]
    vocab = s.weight.shape[0]
    grad_rows, grad_weight = torch.zeros_like(rows), torch.empty_like(s.weight)
    for v in range(0, vocab, PIECE):
        w = s.weight[v:v + PIECE].float()
        x, slope = _capped(s, rows, w)
        p = torch.exp(x - norms[:, None])
        at = targets - v
        here = ((at >= 0) & (at < w.shape[0])).nonzero().flatten()
        p[here, at[here]] -= 1.0
        p *= scale[:, None]
        if slope is not None:
            p *= slope
        grad_rows += p @ w
        grad_weight[v:v + PIECE] = (p.T @ rows).to(grad_weight.dtype)
    grad_hidden = torch.zeros_like(s.hidden)
    grad_hidden[used] = grad_rows.to(grad_hidden.dtype)
    return dict(out, grad_hidden=grad_hidden, grad_weight=grad_weight)


def _plain_logits(s):
    vocab, width = s.codes.shape[0], 2 * s.codes.shape[1]
    x = s.hidden.float()
    out = torch.empty((x.shape[0], vocab), dtype=s.out, device=s.dev)
    for v in range(0, vocab, PIECE):
        c = s.codes[v:v + PIECE]
        q = torch.stack([c & 15, c >> 4], dim=2).view(c.shape[0], width // s.group, s.group).float()
        zero = 8.0 if s.zeros is None else s.zeros[v:v + PIECE].float()[:, :, None]
        w = (q - zero) * s.scales[v:v + PIECE].float()[:, :, None]
        out[:, v:v + PIECE] = (x @ w.view(c.shape[0], width).T).to(s.out)
    return out


# ---- the framework's operators -------------------------------------------------------------------------

_handle = None


def _sampler():
    """The program's one library handle."""
    global _handle
    if _handle is None:
        from opentail.stingray_b200 import BatchSampler

        _handle = BatchSampler(max_rows=MAX_ROWS, max_vocab=LONG, max_history=1, max_top_k=1)
    return _handle


def _own(s):
    b = _sampler()
    if s.kind == "logits":
        s.kept = b.head_logits(s.hidden, s.packed, dtype=s.out, out=s.kept)
        return s.kept
    if s.kept is None:
        s.kept = [None, None]
    s.kept[0] = b.head_loss(s.hidden, s.weight, s.targets, softcap=s.softcap, out=s.kept[0])
    if s.kind == "score":
        return s.kept[0]
    s.kept[1] = b.head_loss_backward(s.hidden, s.weight, s.targets, s.kept[0]["log_norms"], s.grad_loss, softcap=s.softcap, out=s.kept[1])
    return {**s.kept[0], **s.kept[1]}


def run(s):
    if own:
        return _own(s)
    return {"score": _plain_loss, "train": _plain_train, "logits": _plain_logits}[s.kind](s)


# ---- what a pass cannot do without, and what it returns in 64 bits ---------------------------------------

def work(case):
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    if case["kind"] == "logits":
        per_group = 2 * (2 if case["zeros"] else 1)
        weight = vocab * width // 2 + vocab * (width // case["group"]) * per_group
        return {"bytes": weight + rows * width * 2 + rows * vocab * (4 if case["out"] == "f32" else 2), "flops": 2 * rows * width * vocab}
    used = rows - _ignored(case)
    one = used * width * vocab * 2
    read = (used + vocab) * width * 2 + rows * 4
    if case["kind"] == "score":
        return {"bytes": read + rows * 8, "flops": one}
    # three products: the logits, and two with their gradient.  (Not keeping the logits takes a fourth.)
    return {"bytes": read + rows * 12 + (rows + vocab) * width * 2, "flops": 3 * one}


def exact(case, seed):
    s = prepare(case, seed)
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    step = max(256, 2 ** 28 // max(rows, width))  # vocabulary entries of a piece
    if s.kind == "logits":
        h, parts = s.hidden.double(), []
        for v in range(0, vocab, step):
            codes = s.codes[v:v + step].long()
            w = torch.empty((codes.shape[0], width), dtype=torch.float64, device=s.dev)
            w[:, 0::2], w[:, 1::2] = codes % 16, codes // 16
            w -= 8.0 if s.zeros is None else s.zeros[v:v + step].double().repeat_interleave(s.group, 1)
            w *= s.scales[v:v + step].double().repeat_interleave(s.group, 1)
            parts.append(torch.einsum("rd,vd->rv", h, w))
        return torch.cat(parts, 1)
    on = s.targets >= 0
    h = torch.where(on[:, None], s.hidden.double(), 0.0)
    t = s.targets.long().clamp(min=0)
    pieces = [(v, min(vocab, v + step)) for v in range(0, vocab, step)]

    def logits(lo, hi):
        x = torch.einsum("rd,vd->rv", h, s.weight[lo:hi].double())
        return s.softcap * torch.tanh(x / s.softcap) if s.softcap else x

    norm = torch.stack([torch.logsumexp(logits(lo, hi), 1) for lo, hi in pieces], 1).logsumexp(1)
    picked = (h * s.weight[t].double()).sum(1)
    if s.softcap:
        picked = s.softcap * torch.tanh(picked / s.softcap)
    out = {"loss": torch.where(on, norm - picked, 0.0), "log_norms": torch.where(on, norm, 0.0)}
    if s.kind == "score":
        return out
    scale = torch.where(on, s.grad_loss.double(), 0.0)
    of_hidden = torch.zeros((rows, width), dtype=torch.float64, device=s.dev)
    of_weight = torch.empty((vocab, width), dtype=torch.float32, device=s.dev)  # 64 bits do not fit three times; 32 are far below the outputs' 16
    for lo, hi in pieces:
        z = logits(lo, hi)
        d = torch.exp(z - norm[:, None]) - (t[:, None] == torch.arange(lo, hi, device=s.dev)).double()
        d *= scale[:, None]
        if s.softcap:
            d *= 1.0 - (z / s.softcap).square()
        of_hidden += torch.einsum("rv,vd->rd", d, s.weight[lo:hi].double())
        of_weight[lo:hi] = torch.einsum("rv,rd->vd", d, h).float()
    return dict(out, grad_hidden=of_hidden, grad_weight=of_weight)
