"""Head calls issued behind one another without a wait: what one writes - packed weights, factors and hidden states in a workspace that the next
call is given again, gradients that are the next call's hidden states - is what the next one reads."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=4, max_vocab=64, max_history=1, max_top_k=1)
    yield b
    b.close()


def _weight(vocab, width, group, seed, zeros=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = torch.randint(0, 256, (vocab, width // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = ((torch.rand((vocab, width // group), generator=g, device="cuda") - 0.3) / math.sqrt(width)).to(torch.float16)
    z = (torch.rand((vocab, width // group), generator=g, device="cuda") * 20 - 2).to(torch.float16) if zeros else None
    return c, s, z


@pytest.mark.parametrize("rows", [1, 2, 12, 40, 100, 300])
def test_magnitudes_that_change_from_call_to_call(bs, rows):
    """Powers of two times the same hidden states: the logits are the same times them, bit for bit, though rows are scaled by another factor
    every time, which lies at the same address of a workspace."""
    c, s, z = _weight(3000, 512, 64, 1)
    head = bs.head_pack(c, s, z)
    h = torch.randn((rows, 512), generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda").to(torch.bfloat16)
    want = bs.head_logits(h, head)
    powers = [0, 9, -7, 30, -31, 3, 60, -60] * 4
    inputs = [(h.float() * 2.0 ** p).to(torch.bfloat16) for p in powers]
    torch.cuda.synchronize()
    got = [bs.head_logits(x, head) for x in inputs]
    for p, x in zip(powers, got):
        assert torch.equal(x.double(), want.double() * 2.0 ** p), p


@pytest.mark.parametrize("rows", [1, 12, 40, 300])
def test_logits_right_behind_packing(bs, rows):
    weights = [_weight(1000, 256, 32, seed) for seed in range(8)]
    h = torch.randn((rows, 256), generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda").to(torch.float16)
    want = []
    for w in weights:
        head = bs.head_pack(*w)
        torch.cuda.synchronize()
        want.append(bs.head_logits(h, head))
        torch.cuda.synchronize()
    for _ in range(4):
        got = [bs.head_logits(h, bs.head_pack(*w)) for w in weights]  # a packed weight's memory is the next one's
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows", [3, 100, 300])
def test_gradients_as_the_next_call_s_hidden_states(bs, rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = (torch.randn((3000, 256), generator=g, device="cuda") / 16).to(torch.bfloat16)
    h = torch.randn((rows, 256), generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, 3000, (rows,), generator=g, device="cuda", dtype=torch.int32)
    dl = torch.ones(rows, device="cuda")
    head = bs.head_pack(*_weight(3000, 256, 32, 5))

    def chain(wait):
        x, out = h, []
        for _ in range(6):
            f = bs.head_loss(x, w, t)
            wait()
            x = bs.head_loss_backward(x, w, t, f["log_norms"], dl)["grad_hidden"]
            wait()
            out += [f["loss"], x, bs.head_logits(x, head)]
            wait()
        torch.cuda.synchronize()
        return out

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), want))
