"""Losses of rows whose target is certain, and of rows with logits of any size: never below 0, and exact where they are known by heart."""
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


@pytest.mark.parametrize("softcap", [0.0, 70.0])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,width,vocab", [(100, 64, 1000), (700, 256, 3001), (300, 2056, 1000)])
def test_certain_targets_have_no_negative_loss(bs, rows, width, vocab, dtype, softcap):
    """Logits of 5 to 60 for the target, N(0, 0.1^2) for the others."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = torch.randn((vocab, width), generator=g, device="cuda") * 0.1 / math.sqrt(width)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    w = w.to(getattr(torch, dtype))
    lean = torch.linspace(5, 60, rows, device="cuda")[:, None] / w[t.long()].float().square().sum(1, keepdim=True)
    h = (lean * w[t.long()].float()).to(w.dtype)
    f = bs.head_loss(h, w, t, softcap=softcap)
    z = h.double() @ w.double().T
    if softcap:
        z = torch.tanh(z / softcap) * softcap
    want = torch.logsumexp(z, 1) - z.gather(1, t.long()[:, None])[:, 0]
    assert (f["loss"] >= 0).all(), f["loss"].min().item()
    assert (want < 1e-6).sum() > rows / 4  # the case is what it says
    # of the terms beside the target's: logits' differences (1 % for the exponentials' curvature) and the exponentials' 1e-5; and up to 32 of them
    # added to the largest in 32 bits
    off = O.product_bound(h.double(), w.double()).amax(1) + (2.0 ** -19 * z.abs().amax(1) if softcap else 0.0)
    bound = (1 - torch.exp(-want)) * 2.02 * off + 1e-5 * want + 2.0 ** -18
    assert ((f["loss"].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("size", [1.0, 1e4, 3e7, 1e12, 1e30])
@pytest.mark.parametrize("rows,same", [(3, 1), (70, 5), (200, 300)])
def test_equal_logits_of_any_size(bs, rows, same, size):
    """A vocabulary of equal entries: the loss is log(entries) whatever the logits' size; of one entry exactly 0."""
    g = torch.Generator(device="cuda").manual_seed(7)
    row = torch.randn(64, generator=g, device="cuda")
    w = (row * math.sqrt(size)).to(torch.bfloat16).expand(same, 64).contiguous()
    h = (torch.rand((rows, 1), generator=g, device="cuda") + 0.5) * row * math.sqrt(size)
    h[::2] *= -1
    t = torch.arange(rows, device="cuda", dtype=torch.int32) % same
    loss = bs.head_loss(h.to(torch.bfloat16), w, t)["loss"].double()
    if same == 1:
        assert (loss == 0).all()
    # exponentials of 0 are 1; the logarithm and the difference in 64 bits, the loss rounded once
    assert ((loss - math.log(same)).abs() <= math.log(same) * 2.0 ** -23).all(), (loss - math.log(same)).abs().max().item()
