"""Soft caps of the head's losses over their whole range: against the formula in 64 bits, with an error that is relative to the
logit and not to the cap.

cap * tanh(z / cap) is off by its own arithmetic by less than 2^-19 of itself: with x = z / cap 2^-23 off, a series in x^2 below
|x| = 1/4 (its first omitted term 2^-26.8, three roundings that count: 2^-22), and 1 - 2 q, q = 1 / (exp(2 x) + 1), above: an exponential 2^-22 (1 + 2 x) off
(its own 2^-22, its argument's), a reciprocal and a sum 2^-22.4 off make 2 q (e / (e + 1) (1 + 2 x) + 0.76) 2^-22, which is 5.5 * 2^-22 of
tanh(1/4) and less behind it."""
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


class Capped(O.Loss):
    """The oracle's losses and gradients; of a capped logit 2^-19 is the function's own."""

    def __init__(self, hidden, weight, targets, softcap):
        super().__init__(hidden, weight, targets)
        z = self.h @ self.w.T
        th = torch.tanh(z / softcap)
        # small arguments in 64 bits: tanh(x) cap is z (1 - x^2 / 3) where nothing else of it is left
        self.z = torch.where((z / softcap).abs() < 1e-5, z * (1 - (z / softcap) ** 2 / 3), th * softcap)
        self.slope, self.softcap = 1 - th * th, softcap
        self.dz = self.dz + self.z.abs() * 2.0 ** -19
        n = self.z.logsumexp(1)
        most = self.dz.amax(1)
        self.norm, self.d_norm = n, most + 1e-5 + n.abs() * 2.0 ** -23
        picked = self.z.gather(1, self.t[:, None])[:, 0]
        self.log_norms[self.on], self.loss[self.on] = n, n - picked
        self.d_norms[self.on] = self.d_norm
        self.d_loss[self.on] = self.d_norm + most + (n - picked).abs() * 2.0 ** -23


def _inputs(rows, width, vocab, dtype, seed=0, std=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + 31 * width + 977 * vocab)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (std / math.sqrt(width))).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    h = (torch.randn((rows, width), generator=g, device="cuda") + w[t.long()].float()).to(dtype)
    return h, w, t, torch.rand(rows, generator=g, device="cuda") * 2 - 0.5


def _near(name, got, want, bound):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    assert (off <= bound).all(), f"{name}: {off.max().item():.3g} off, {(off - bound).max().item():.3g} above the bound"


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,width,vocab", [(20, 64, 900), (150, 136, 3001)])
@pytest.mark.parametrize("cap", [0.5, 5.0, 30.0, 100.0, 1e4, 1e6, 1e8, 1e30, 2.9e38])
def test_caps_of_every_size(bs, cap, rows, width, vocab, dtype):
    h, w, t, dl = _inputs(rows, width, vocab, getattr(torch, dtype))
    cap = torch.tensor(cap).item()  # as the library is given it
    want = Capped(h, w, t, cap)
    f = bs.head_loss(h, w, t, softcap=cap)
    _near("loss", f["loss"], want.loss, want.d_loss)
    _near("log_norms", f["log_norms"], want.log_norms, want.d_norms)
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl, softcap=cap)
    gh, dh, gw, dw = want.grads(dl)
    _near("grad_hidden", b["grad_hidden"], gh, dh)
    _near("grad_weight", b["grad_weight"], gw, dw)


@pytest.mark.parametrize("std", [1e-3, 0.3, 30.0])
def test_one_logit_at_a_time(bs, std):
    """Two vocabulary entries, one of them with the logit 0: the loss of that one is log(1 + exp(c)) of the capped logit c, whose slope
    is at most 1, so errors of c show as they are."""
    g = torch.Generator(device="cuda").manual_seed(11)
    h = (torch.randn((128, 8), generator=g, device="cuda") * std).to(torch.float16)
    w = torch.zeros((2, 8), dtype=torch.float16, device="cuda")
    w[1, 0] = 1
    t = torch.zeros(128, dtype=torch.int32, device="cuda")
    for cap in (0.1, 1.0, 30.0, 1e3, 1e5, 1e9):
        x = h[:, 0].double()
        c = torch.where((x / cap).abs() < 1e-5, x * (1 - (x / cap) ** 2 / 3), cap * torch.tanh(x / cap))
        want = torch.logaddexp(c, torch.zeros_like(c))
        off = (bs.head_loss(h, w, t, softcap=cap)["loss"].double() - want).abs()
        # the exponentials and the logarithm of their sum: 2^-21; the loss as a difference in 32 bits
        assert (off <= c.abs() * 2.0 ** -19 + 2.0 ** -21 + want * 2.0 ** -22).all(), (cap, (off / (1 + c.abs())).max().item())
