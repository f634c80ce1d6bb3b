"""Gradients of rows with logits of any size, whose largest alone counts: probabilities of exactly 1 and 0."""
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


@pytest.mark.parametrize("rows", [20, 100, 200])
@pytest.mark.parametrize("dtype,size", [("bfloat16", 1e3), ("bfloat16", 1e5), ("bfloat16", 3e7), ("bfloat16", 1e12), ("bfloat16", 1e30), ("float16", 1e3), ("float16", 1e5)])
def test_certain_rows_of_any_size(bs, size, rows, dtype):
    """Vocabulary entries are 1 .. 4 times one direction, hidden states plus or minus it: the fourth entry or the first is certain."""
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(rows)
    one = torch.sign(torch.randn(64, generator=g, device="cuda")) * size ** 0.5 / 8  # 64 products of size / 64
    w = (torch.arange(1, 5, device="cuda").float()[:, None] * one).to(dtype)
    sign = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    h = (sign[:, None] * one).to(dtype)
    t = torch.randint(0, 4, (rows,), generator=g, device="cuda", dtype=torch.int32)
    dl = torch.randint(2, 6, (rows,), generator=g, device="cuda").float() / 4  # 16 bits hold them
    n = bs.head_loss(h, w, t)["log_norms"]
    z = h.double() @ w.double().T
    assert (z.sort(1, descending=True).values.diff(dim=1).abs().amin() > 200).all()
    b = bs.head_loss_backward(h, w, t, n, dl)
    best = z.argmax(1)
    p = torch.nn.functional.one_hot(best, 4).double() - torch.nn.functional.one_hot(t.long(), 4).double()
    p *= dl.double()[:, None]
    for got, want, size_of in ((b["grad_hidden"], p @ w.double(), p.abs() @ w.double().abs()), (b["grad_weight"], p.T @ h.double(), p.abs().T @ h.double().abs())):
        bound = want.abs() * O.U[dtype] + (rows / 16 + 4) * O.STEP * size_of
        assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all()
    assert (b["grad_hidden"][best == t] == 0).all()
