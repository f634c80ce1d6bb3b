"""Gradients whose sums are long: wide hidden states, and many rows.  They are as far off as their own rounding, which is evenly spread below half a
step - 0.29 steps of 2 U relative to the value's power of two, 0.58 U of the value at worst - also where every term has one sign, or a row's
likeliest token is a wrong one: fp16, whose rounding is the smaller."""
import math

import pytest
import torch

from tests import head_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=4, max_vocab=64, max_history=1, max_top_k=1)
    yield b
    b.close()


def _grads(h, w, t, dl, n):
    """The gradients in 64 bits, over slices of the rows."""
    gh, gw = [], torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    for lo in range(0, h.shape[0], 8192):
        hh, tt, on = h[lo:lo + 8192].double(), t[lo:lo + 8192].long(), (t[lo:lo + 8192] >= 0).double()
        g = torch.softmax(hh @ w.double().T, 1)
        g.scatter_add_(1, tt.clamp(min=0)[:, None], -torch.ones_like(g[:, :1]))
        g *= (dl[lo:lo + 8192].double() * on)[:, None]
        gh.append(g @ w.double())
        gw += g.T @ hh
    return torch.cat(gh), gw


def _off(got, want):
    return ((got.double() - want).norm() / want.norm()).item() / O.U[got.dtype]


@pytest.mark.parametrize("certain", [2.0, 9.0])
@pytest.mark.parametrize("rows,width,vocab", [(20, 16_384, 2000), (200, 12_296, 2000), (20, 65_536, 300), (100, 8200, 1000), (150, 4104, 1000)])
def test_wide_rows_with_a_likely_wrong_token(bs, rows, width, vocab, certain):
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2.5 / math.sqrt(width))).to(torch.float16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    wrong = (t.long() + 1 + torch.randint(0, vocab - 1, (rows,), generator=g, device="cuda")) % vocab
    h = (torch.randn((rows, width), generator=g, device="cuda") + certain * w[wrong].float()).to(torch.float16)  # a logit 6.25 times it
    n = bs.head_loss(h, w, t)["log_norms"]
    dl = torch.ones(rows, device="cuda")
    b = bs.head_loss_backward(h, w, t, n, dl)
    gh, gw = _grads(h, w, t, dl, n)
    assert _off(b["grad_hidden"], gh) <= 0.58 and _off(b["grad_weight"], gw) <= 0.58


@pytest.mark.parametrize("softcap", [0.0, 40.0])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,width,vocab", [(60, 4104, 700), (300, 5000, 513), (70, 16_400, 1000), (140, 17_000, 300)])
def test_wide_rows_within_the_oracle_s_bounds(bs, rows, width, vocab, dtype, softcap):
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2.5 / math.sqrt(width))).to(getattr(torch, dtype))
    t = torch.randint(-100, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    h = torch.randn((rows, width), generator=g, device="cuda").to(w.dtype)
    dl, dn = torch.rand(rows, generator=g, device="cuda") - 0.3, torch.randn(rows, generator=g, device="cuda") * 0.1
    want = O.Loss(h, w, t, softcap)
    f = bs.head_loss(h, w, t, softcap=softcap)
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl, grad_log_norms=dn, softcap=softcap)
    gh, dh, gw, dw = want.grads(dl, dn)
    assert ((b["grad_hidden"].double() - gh).abs() <= dh).all() and ((b["grad_weight"].double() - gw).abs() <= dw).all()
    again = bs.head_loss_backward(h, w, t, f["log_norms"], dl, grad_log_norms=dn, softcap=softcap)
    assert all(torch.equal(again[k], b[k]) for k in b)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows,width,vocab", [(16_385, 72, 700), (70_000, 72, 130), (262_100, 200, 130), (20_000, 64, 15_001)])
def test_many_rows_of_one_sign(bs, rows, width, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2.5 / math.sqrt(width))).to(getattr(torch, dtype))
    h = torch.randn((rows, width), generator=g, device="cuda").abs().to(w.dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    t[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1
    dl = torch.full((rows,), 2.0 ** -6, device="cuda")
    n = bs.head_loss(h, w, t)["log_norms"]
    b = bs.head_loss_backward(h, w, t, n, dl)
    gh, gw = _grads(h, w, t, dl, n)
    assert _off(b["grad_weight"], gw) <= 0.58
    # of hidden states beyond 64 rows the roundings of a row's other probabilities remain: below a third of a step of theirs, added to its own
    assert _off(b["grad_hidden"], gh) <= 0.58 + 0.33
    again = bs.head_loss_backward(h, w, t, n, dl, want_hidden=False)
    assert torch.equal(again["grad_weight"], b["grad_weight"])


@pytest.mark.parametrize("mean", [1.0, 4.0])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows,width,vocab", [(60, 72, 200_001), (100, 512, 262_144), (300, 264, 150_000), (1000, 512, 131_072), (1000, 2048, 40_000), (20, 1032, 40_000)])
def test_weights_with_a_mean(bs, rows, width, vocab, dtype, mean):
    """A direction that all vocabulary entries share: of the sums over the vocabulary that is most, and a row's target takes it off again, so that it is
    the probabilities' sum that shows, and every addition."""
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    s = 2.5 / math.sqrt(width)
    w = ((torch.randn((vocab, width), generator=g, device="cuda") + mean) * s).to(getattr(torch, dtype))
    h = torch.randn((rows, width), generator=g, device="cuda").to(w.dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    n = bs.head_loss(h, w, t)["log_norms"]
    one = torch.ones(rows, device="cuda")
    b = bs.head_loss_backward(h, w, t, n, one, want_weight=False)["grad_hidden"]
    norm = torch.stack([torch.logsumexp(h.double() @ w[v:v + 16384].double().T, 1) for v in range(0, vocab, 16384)], 1).logsumexp(1)
    gh = -w[t.long()].double()
    for v in range(0, vocab, 16384):
        x = w[v:v + 16384].double()
        gh += torch.exp(h.double() @ x.T - norm[:, None]) @ x
    # beyond 64 rows the roundings of the other probabilities remain, as above; and a part's additions, 1024 at most (bf16: 8192), are off by 2^-22 of the
    # sum each: U / 2 of the probabilities' products with the weight's sizes
    sizes = sum(torch.exp(h.double() @ w[v:v + 16384].double().T - norm[:, None]) @ w[v:v + 16384].double().abs() for v in range(0, vocab, 16384))
    assert _off(b, gh) <= 0.58 + (0.33 if rows > 64 else 0.0) + 0.5 * (sizes.norm() / gh.norm()).item()
    assert torch.equal(bs.head_loss_backward(h, w, t, n, one, want_weight=False)["grad_hidden"], b)


def test_small_probabilities_beside_a_large_target(bs):
    """Probabilities of 1 / 40,000 each, weights of 1, and of 200 for the targets, the vocabulary's first: what the 40,000 add up to is 1.02, of
    which nothing is lost beside the target's 200."""
    w = torch.ones((40_000, 2048), dtype=torch.float16, device="cuda")
    w[:4] = 200
    h = torch.zeros((3000, 2048), dtype=torch.float16, device="cuda")
    t = (torch.arange(3000, device="cuda") % 4).to(torch.int32)
    n = bs.head_loss(h, w, t)["log_norms"]
    b = bs.head_loss_backward(h, w, t, n, torch.ones(3000, device="cuda"), want_weight=False)["grad_hidden"]
    want = (39_996 + 4 * 200) / 40_000 - 200
    # half a step of fp16 at 199; the probability's rounding and the sums' additions 2^-12 of 1.02 each, the normaliser's 2^-22
    assert ((b.double() - want).abs() <= 0.0625 + 2 * 1.02 * 2.0 ** -12 + 1e-5).all(), (b.double() - want).abs().max().item()
