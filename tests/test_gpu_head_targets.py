"""Gradients of rows that share targets as the tokens of a text do: a few targets with very many rows, many with a few, all rows with one.  Against
the formulas in 64 bits; the tolerances are head_oracle's."""
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


def _inputs(rows, width, vocab, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + vocab)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2.5 / math.sqrt(width))).to(dtype)
    h = torch.randn((rows, width), generator=g, device="cuda").to(dtype)
    return g, h, w, torch.rand(rows, generator=g, device="cuda") * 2 - 0.5


def _check(bs, h, w, t, dl):
    want = O.Loss(h, w, t)
    f = bs.head_loss(h, w, t)
    assert ((f["loss"].double() - want.loss).abs() <= want.d_loss).all()
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl)
    gh, dh, gw, dw = want.grads(dl)
    for name, x, y, bound in (("grad_hidden", b["grad_hidden"], gh, dh), ("grad_weight", b["grad_weight"], gw, dw)):
        off = (x.double() - y).abs()
        assert torch.isfinite(x).all() and (off <= bound).all(), (name, off.max().item(), (off - bound).max().item())
    again = bs.head_loss_backward(h, w, t, f["log_norms"], dl)
    assert all(torch.equal(again[k], b[k]) for k in b)
    return b, gw


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,width,vocab", [(3000, 72, 1000), (5000, 200, 513), (700, 1032, 300)])
def test_targets_as_in_a_text(bs, rows, width, vocab, dtype):
    """The k-th token 1 / k as often as the first, the frequent ones next to one another."""
    g, h, w, dl = _inputs(rows, width, vocab, getattr(torch, dtype), 1)
    p = 1.0 / torch.arange(1, vocab + 1, device="cuda").float()
    t = torch.multinomial(p, rows, replacement=True, generator=g).to(torch.int32)
    t[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1
    _check(bs, h, w, t, dl)


@pytest.mark.parametrize("counts", [[5], [33, 1, 2], [4, 5, 6, 7], [31, 32, 33, 64, 65], [1500, 3, 1, 40] * 8, [2000] + [5] * 40, [20] * 64])
def test_runs_of_every_length(bs, counts):
    """So many rows of each of these targets, one target after the other, rows shuffled; and rows with targets of their own beside them."""
    rows, width, vocab = sum(counts) + 100, 136, 400
    g, h, w, dl = _inputs(rows, width, vocab, torch.bfloat16, 2)
    t = torch.cat([torch.full((n,), 37 + i, dtype=torch.int32) for i, n in enumerate(counts)] + [torch.arange(300, 400, dtype=torch.int32)]).cuda()
    t = t[torch.randperm(rows, generator=g, device="cuda")].contiguous()
    _check(bs, h, w, t, dl)


@pytest.mark.parametrize("rows,width,vocab,target", [(66, 64, 700, 699), (8192, 64, 300, 0), (40_000, 24, 5, 3)])
def test_all_rows_have_one_target(bs, rows, width, vocab, target):
    _, h, w, dl = _inputs(rows, width, vocab, torch.bfloat16, 3)
    t = torch.full((rows,), target, dtype=torch.int32, device="cuda")
    _check(bs, h, w, t, dl)


def test_rows_in_another_order(bs):
    """The targets' gradients are added in the order of the rows, whatever it is: the same rows in another one are as close to the formula."""
    g, h, w, dl = _inputs(2000, 64, 50, torch.bfloat16, 4)
    t = (torch.arange(2000, device="cuda") % 3).to(torch.int32)
    one, want = _check(bs, h, w, t, dl)
    turn = torch.randperm(2000, generator=g, device="cuda")
    two, _ = _check(bs, h[turn].contiguous(), w, t[turn].contiguous(), dl[turn].contiguous())
    for b in (one, two):  # nearly their own rounding, evenly spread below half a step: 0.29 steps of 2 U, 0.58 U of the value at worst
        assert ((b["grad_weight"].double() - want).norm() / want.norm()).item() <= 0.58 * O.U[torch.bfloat16]


def test_as_many_rows_as_there_may_be_with_one_target(bs):
    """2^20 rows, of which a bounded wait of the products must not run out."""
    rows = 1 << 20
    _, h, w, dl = _inputs(rows, 8, 3, torch.bfloat16, 5)
    t = torch.full((rows,), 1, dtype=torch.int32, device="cuda")
    t[::5] = -1
    _check(bs, h, w, t, dl)
