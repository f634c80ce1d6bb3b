"""stg_head_pack and stg_head_logits against the formula in 64 bits; the tolerances are head_oracle's, and a rounding of bf16 logits."""
import math

import pytest

from tests import head_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=32, max_vocab=5000, max_history=8, max_top_k=64)
    yield b
    b.close()


def _inputs(rows, width, vocab, group, dtype, scales, zeros, seed=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed + rows + 31 * width + 977 * vocab + group)
    h = torch.randn((rows, width), generator=g, device="cuda").to(dtype)
    c = torch.randint(0, 256, (vocab, width // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = ((torch.rand((vocab, width // group), generator=g, device="cuda") - 0.3) / math.sqrt(width)).to(scales)
    z = (torch.rand((vocab, width // group), generator=g, device="cuda") * 20 - 2).to(scales) if zeros else None
    return h, c, s, z


def _check(got, h, c, s, z):
    import torch

    want, bound = O.logits(h, c, s, z)
    if got.dtype == torch.bfloat16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"{off.max().item():.3g} off, {(off - bound).max().item():.3g} above the bound"


SIZES = [(1, 32, 1, 32), (1, 64, 15, 32), (1, 96, 16, 32), (2, 128, 17, 64), (7, 128, 127, 128), (8, 192, 128, 64), (9, 160, 129, 32), (16, 256, 1000, 128),
         (17, 2048, 333, 64), (1, 4096, 4001, 128), (31, 2080, 500, 32), (33, 1024, 2000, 128), (64, 4224, 257, 128), (65, 512, 1025, 32), (128, 640, 700, 128),
         (200, 320, 3001, 64), (256, 896, 2048, 64), (300, 1152, 130, 128), (1, 65_536, 40, 32)]


@pytest.mark.parametrize("dtype,scales,zeros,out", [("bfloat16", "float16", False, "float32"), ("bfloat16", "bfloat16", True, "bfloat16"),
                                                    ("float16", "float16", True, "float32"), ("float16", "bfloat16", False, "bfloat16")])
@pytest.mark.parametrize("rows,width,vocab,group", SIZES)
def test_logits(bs, rows, width, vocab, group, dtype, scales, zeros, out):
    import torch

    h, c, s, z = _inputs(rows, width, vocab, group, getattr(torch, dtype), getattr(torch, scales), zeros)
    head = bs.head_pack(c, s, z)
    assert (head.vocab, head.width, head.group, head.has_zeros) == (vocab, width, group, zeros)
    _check(bs.head_logits(h, head, dtype=getattr(torch, out)), h, c, s, z)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_every_code(bs, dtype):
    """One hidden state per column: the weight comes back, every code of every place in a group."""
    import torch

    width, vocab = 128, 64
    c = torch.arange(vocab * width // 2, device="cuda").view(vocab, width // 2).mul(37).add(11).remainder(256).to(torch.uint8)
    s = torch.ones((vocab, width // 32), dtype=torch.float16, device="cuda")
    h = torch.eye(width, dtype=getattr(torch, dtype), device="cuda")
    got = bs.head_logits(h, bs.head_pack(c, s))
    w, _ = O.unpack(c, s, None)
    assert torch.equal(got.T.double(), w)


@pytest.mark.parametrize("rows", [1, 5, 20, 40])
def test_strides_and_places_behind(bs, rows):
    """Rows of hidden states, codes and logits inside wider ones: what lies behind is neither read nor written."""
    import torch

    h, c, s, z = _inputs(rows, 192, 1001, 64, torch.bfloat16, torch.float16, True)
    ref = bs.head_logits(h, bs.head_pack(c, s, z))
    codes = torch.full((1001, 131), 255, dtype=torch.uint8, device="cuda")
    codes[:, 3:99] = c
    head = bs.head_pack(codes[:, 3:99], s, z)
    for shift in (0, 1, 8):
        wide = torch.full((rows, 215), float("nan"), dtype=h.dtype, device="cuda")
        wide[:, shift:shift + 192] = h
        for dtype in (torch.float32, torch.bfloat16):
            room = torch.full((rows + 2, 1009), 7.0, dtype=dtype, device="cuda")
            view = room[1:rows + 1, 1:1002]
            assert bs.head_logits(wide[:, shift:shift + 192], head, out=view) is view
            assert torch.equal(view, ref.to(dtype))
            assert (room[[0, rows + 1]] == 7).all() and (room[:, 0] == 7).all() and (room[:, 1002:] == 7).all()


@pytest.mark.parametrize("rows", [3, 40, 140])
def test_rows_do_not_depend_on_one_another(bs, rows):
    """A row that is not finite changes no other row; scales that are not finite no other column."""
    import torch

    h, c, s, z = _inputs(rows, 256, 600, 64, torch.float16, torch.float16, True)
    ref = bs.head_logits(h, bs.head_pack(c, s, z))
    h[1, 7] = float("nan")
    s[300, 1] = float("inf")
    got = bs.head_logits(h, bs.head_pack(c, s, z))
    assert torch.isnan(got[1]).all() and not torch.isfinite(got[:, 300]).any()
    keep = torch.ones(600, dtype=torch.bool, device="cuda")
    keep[300] = False
    rest = torch.arange(rows, device="cuda") != 1
    assert torch.equal(got[rest][:, keep], ref[rest][:, keep])


def test_no_rows(bs):
    import torch

    h, c, s, _ = _inputs(4, 64, 100, 32, torch.bfloat16, torch.float16, False)
    assert bs.head_logits(h[:0], bs.head_pack(c, s)).shape == (0, 100)


@pytest.mark.parametrize("rows", [1, 12, 100])
def test_repeats_streams_and_graphs(bs, rows):
    import torch

    h, c, s, z = _inputs(rows, 512, 5000, 64, torch.bfloat16, torch.float16, True)
    h2 = _inputs(rows, 512, 5000, 64, torch.bfloat16, torch.float16, True, seed=9)[0]
    head = bs.head_pack(c, s, z)
    want, want2 = bs.head_logits(h, head), bs.head_logits(h2, head)
    assert torch.equal(bs.head_logits(h, head), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [bs.head_logits(x, head, stream=streams[i % 2]) for i, x in enumerate((h, h2, h, h2))]
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, (want, want2, want, want2)))
    graphs, x = [], h.clone()
    for st in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            o = bs.head_logits(x, head)
        graphs.append((g, st, o))
    x.copy_(h2)
    torch.cuda.synchronize()
    for g, st, _ in graphs * 2:
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want2) for _, _, o in graphs)


def test_decode_score_train(bs):
    """The head as a program uses it: logits in 4 bits, a token per row sampled from them and by beams, the tokens' losses
    from the unpacked weight, and a step down the gradient."""
    import numpy as np
    import torch
    from opentail.stingray_b200 import SamplingParams

    rows, width, vocab = 8, 256, 5000
    h, c, s, z = _inputs(rows, width, vocab, 64, torch.bfloat16, torch.bfloat16, True)
    logits = bs.head_logits(h, bs.head_pack(c, s, z))
    got = bs.sample_rows(logits, [SamplingParams(Temperature=0.0)] * rows, want_flags=True)
    assert torch.equal(got["tokens"].long(), logits.argmax(1))
    drawn = bs.sample_rows(logits, [SamplingParams(TopK=40)] * rows, uniforms=np.linspace(0.05, 0.95, rows).astype(np.float32))["tokens"]
    best = bs.beam_select(logits, torch.zeros((2, 4), device="cuda"), 8, want_norms=True)
    weight = O.unpack(c, s, z)[0].to(torch.bfloat16)
    f = bs.head_loss(h, weight, drawn)
    want = O.Loss(h, weight, drawn)
    assert ((f["loss"].double() - want.loss).abs() <= want.d_loss).all()
    # the beams' normalisers are those of the unrounded weight: a weight's rounding moves a logit by 2^-8 of its terms' sizes
    moved = 2.0 ** -8 * (h.double().abs() @ weight.double().abs().T).amax(1)
    assert ((best["log_norms"].flatten().double() - f["log_norms"].double()).abs() <= moved + want.d_norms + 1e-4).all()
    g = bs.head_loss_backward(h, weight, drawn, f["log_norms"], torch.full((rows,), 1.0 / rows, device="cuda"))
    gh, dh, gw, dw = want.grads(torch.full((rows,), 1.0 / rows, device="cuda"))
    assert ((g["grad_hidden"].double() - gh).abs() <= dh).all() and ((g["grad_weight"].double() - gw).abs() <= dw).all()


def test_refusals(bs):
    import torch
    from opentail.stingray_b200 import StingrayError

    h, c, s, z = _inputs(4, 192, 100, 64, torch.bfloat16, torch.float16, True)
    head = bs.head_pack(c, s, z)
    for a in ((c.int(), s, z), (c, s.float(), None), (c, s[:50], None), (c, s, z.bfloat16()), (c, s, z[:, :1]), (c.cpu(), s, z), (c.T, s, z)):
        with pytest.raises(ValueError):
            bs.head_pack(*a)
    wide = torch.ones((100, 12), dtype=torch.float16, device="cuda")
    for scales in (wide, wide[:, :1].contiguous(), wide[:, :2].contiguous()):  # groups of 16, 192 and 96 columns
        with pytest.raises(StingrayError) as e:
            bs.head_pack(c, scales)
        assert e.value.code == 4
    for x in (h.float(), h[:, :128], h.cpu(), h[0]):
        with pytest.raises(ValueError):
            bs.head_logits(x, head)
    for out in (torch.empty((4, 99), device="cuda"), torch.empty((3, 100), device="cuda"), torch.empty((4, 100), dtype=torch.float16, device="cuda"),
                torch.empty((4, 200), device="cuda")[:, ::2]):
        with pytest.raises(ValueError):
            bs.head_logits(h, head, out=out)
    with pytest.raises(ValueError):
        bs.head_logits(h, head, dtype=torch.float16)
