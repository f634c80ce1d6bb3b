"""Losses and gradients of calls that are cut up: several pieces of the vocabulary, the last one short, and more rows of tiles than are taken
as a group.  Against the formulas in 64 bits; the tolerances are head_oracle's."""
import math
import os
import subprocess

import pytest
import torch

from tests import head_oracle as O

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=4, max_vocab=64, max_history=1, max_top_k=1)
    yield b
    b.close()


@pytest.fixture(scope="module")
def pieces():
    """(pieces, entries of a piece) of a backward call, from the plan that the library makes."""
    out = os.path.join(ROOT, "tests", "cpp", "_build", "head_pieces")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "opentail", "stingray_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "head_pieces.cpp"), "-o", out], check=True)
    sms = torch.cuda.get_device_properties(0).multi_processor_count

    def ask(rows, vocab, width):
        r = subprocess.run([out, str(rows), str(vocab), str(width), str(sms)], capture_output=True, text=True, check=True)
        return tuple(int(x) for x in r.stdout.split())

    return ask


class Slice(O.Loss):
    """Some of the rows; ``sizes``: of the terms of the weight's gradient."""

    def _joined(self, g, dg, u):
        self.sizes = g.abs().T @ self.h.abs()
        return super()._joined(g, dg, u)


@pytest.mark.parametrize("dtype,rows,width,vocab,softcap", [("bfloat16", 4200, 64, 33_001, 0.0), ("float16", 4200, 64, 33_001, 30.0), ("bfloat16", 9000, 200, 30_017, 0.0),
                                                            ("float16", 60_000, 16, 4500, 0.0)])
def test_pieces_of_the_vocabulary(bs, pieces, dtype, rows, width, vocab, softcap):
    n, piece = pieces(rows, vocab, width)
    assert n > 1 and vocab % piece != 0 and (n - 1) * piece < vocab
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2.5 / math.sqrt(width))).to(getattr(torch, dtype))
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    # targets on both sides of every boundary, the vocabulary's ends among them, some of them several rows'
    edges = sorted({0, vocab - 1} | {e for i in range(1, n) for e in (i * piece - 1, i * piece)})
    t[:3 * len(edges)] = torch.tensor(edges * 3, dtype=torch.int32, device="cuda")
    h = (torch.randn((rows, width), generator=g, device="cuda") + w[t.long()].float()).to(w.dtype)
    t[torch.rand(rows, generator=g, device="cuda") < 0.2] = -100
    dl, dn = torch.rand(rows, generator=g, device="cuda") * 2 - 0.5, torch.randn(rows, generator=g, device="cuda") * 0.1
    f = bs.head_loss(h, w, t, softcap=softcap)
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl, grad_log_norms=dn, softcap=softcap)

    # the oracle over slices of the rows, whose gradients of the weight add up
    gw, dw = (torch.zeros((vocab, width), dtype=torch.float64, device="cuda") for _ in range(2))
    largest = max(dl[t >= 0].abs().max().item(), (dl + dn)[t >= 0].abs().max().item())
    for lo in range(0, rows, 1500):
        s = slice(lo, lo + 1500)
        want = Slice(h[s], w, t[s], softcap)
        assert ((f["loss"][s].double() - want.loss).abs() <= want.d_loss).all() and ((f["log_norms"][s].double() - want.log_norms).abs() <= want.d_norms).all()
        gh, dh, part, d_part = want.grads(dl[s], dn[s])
        # fp16 ends 2^-37 below the largest factor of all rows, of which the slice knows its own
        rest = largest * 2.0 ** -37 * want.w.abs().sum(0)
        off = (b["grad_hidden"][s].double() - gh).abs()
        assert (off <= dh + rest).all(), (lo, (off - dh - rest).max().item())
        gw += part
        dw += d_part + largest * 2.0 ** -37 * want.h.abs().sum(0) + rows / 16 * O.STEP * want.sizes  # a sum over all rows has their additions
    off = (b["grad_weight"].double() - gw).abs()
    assert torch.isfinite(b["grad_weight"]).all() and (off <= dw).all(), (off - dw).max().item()

    one = bs.head_loss_backward(h, w, t, f["log_norms"], dl, grad_log_norms=dn, softcap=softcap, want_weight=False)
    two = bs.head_loss_backward(h, w, t, f["log_norms"], dl, grad_log_norms=dn, softcap=softcap, want_hidden=False)
    again = bs.head_loss_backward(h, w, t, f["log_norms"], dl, grad_log_norms=dn, softcap=softcap)
    assert torch.equal(one["grad_hidden"], b["grad_hidden"]) and torch.equal(two["grad_weight"], b["grad_weight"])
    assert all(torch.equal(again[k], b[k]) for k in b)


def test_more_rows_of_tiles_than_a_group(bs):
    """4096 rows and more: the logits' tiles are taken in groups of 16 rows of tiles, the last group is not full."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for rows, vocab in ((4097, 600), (5000, 257), (8500, 1000)):
        w = (torch.randn((vocab, 136), generator=g, device="cuda") * 0.2).to(torch.bfloat16)
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        h = torch.randn((rows, 136), generator=g, device="cuda").to(torch.bfloat16)
        want = O.Loss(h, w, t)
        f = bs.head_loss(h, w, t)
        assert ((f["loss"].double() - want.loss).abs() <= want.d_loss).all() and ((f["log_norms"].double() - want.log_norms).abs() <= want.d_norms).all()
        dl = torch.rand(rows, generator=g, device="cuda")
        b = bs.head_loss_backward(h, w, t, f["log_norms"], dl)
        gh, dh, gw, dw = want.grads(dl)
        assert ((b["grad_hidden"].double() - gh).abs() <= dh).all() and ((b["grad_weight"].double() - gw).abs() <= dw).all()
