"""stg_head_loss and stg_head_loss_backward against the formulas in 64 bits; the tolerances are head_oracle's."""
import math

import numpy as np
import pytest

from tests import head_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=4, max_vocab=64, max_history=1, max_top_k=1)  # the head is not bounded by these
    yield b
    b.close()


def _inputs(rows, width, vocab, dtype, seed=0, ignored=0.0, std=2.5):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed + rows + 31 * width + 977 * vocab)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (std / math.sqrt(width))).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    h = (torch.randn((rows, width), generator=g, device="cuda") + w[t.long()].float()).to(dtype)
    t[torch.rand(rows, generator=g, device="cuda") < ignored] = -100
    dl = torch.rand(rows, generator=g, device="cuda") * 2 - 0.5
    dn = torch.randn(rows, generator=g, device="cuda") * 0.1
    return h, w, t, dl, dn


def _near(name, got, want, bound):
    import torch

    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{name}: {off.max().item():.3g} off, {worst:.3g} above the bound"


def _check(bs, h, w, t, dl, dn=None, softcap=0.0):
    want = O.Loss(h, w, t, softcap)
    f = bs.head_loss(h, w, t, softcap=softcap)
    _near("loss", f["loss"], want.loss, want.d_loss)
    _near("log_norms", f["log_norms"], want.log_norms, want.d_norms)
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl, grad_log_norms=dn, softcap=softcap)
    gh, dh, gw, dw = want.grads(dl, dn)
    _near("grad_hidden", b["grad_hidden"], gh, dh)
    _near("grad_weight", b["grad_weight"], gw, dw)
    off = t < 0
    assert (f["loss"][off] == 0).all() and (f["log_norms"][off] == 0).all() and (b["grad_hidden"][off] == 0).all()
    return f, b


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,width,vocab,ignored,softcap,norms", [
    (1, 8, 1, 0, 0, False), (1, 64, 2, 0, 0, True), (3, 72, 255, 0, 0, False), (5, 128, 256, 0, 30, True), (2, 504, 257, 0, 0, False),
    (127, 256, 1000, 0, 0, True), (128, 64, 511, 0.3, 0, False), (129, 520, 4096, 0.1, 5, True), (300, 264, 40_001, 0.6, 0, False), (7, 1032, 33_333, 0, 30, False),
    (513, 384, 2049, 0.5, 0, True), (1, 2048, 50_257, 0, 0, False), (64, 72, 20_000, 0, 0, False), (1100, 96, 3000, 0, 0, False),
])
def test_losses_and_gradients(bs, rows, width, vocab, ignored, softcap, norms, dtype):
    import torch

    h, w, t, dl, dn = _inputs(rows, width, vocab, getattr(torch, dtype), ignored=ignored)
    _check(bs, h, w, t, dl, dn if norms else None, softcap)


def test_longer_sums(bs):
    """Widths and row counts beyond what one accumulator is given at a time."""
    import torch

    h, w, t, dl, _ = _inputs(260, 4104, 700, torch.bfloat16)
    _check(bs, h, w, t, dl)
    h, w, t, dl, _ = _inputs(3000, 64, 600, torch.float16, ignored=0.2)
    _check(bs, h, w, t, dl)


@pytest.mark.parametrize("rows,vocab", [(70, 5), (200, 3), (1500, 40), (2500, 1), (65, 900)])
def test_many_rows_with_one_target(bs, rows, vocab):
    """Rows that share targets: the remainders of their gradients are added up in their order, repeatably."""
    import torch

    h, w, t, dl, dn = _inputs(rows, 72, vocab, torch.bfloat16, ignored=0.1)
    _, b = _check(bs, h, w, t, dl, dn)
    n = bs.head_loss(h, w, t)["log_norms"]
    for _ in range(2):
        b2 = bs.head_loss_backward(h, w, t, n, dl, grad_log_norms=dn)
        assert torch.equal(b["grad_weight"], b2["grad_weight"]) and torch.equal(b["grad_hidden"], b2["grad_hidden"])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 64, 65, 300])
def test_gradients_are_nearly_their_own_rounding(bs, rows, dtype):
    """The roundings of the logits' gradients even out or are made good: both results are about as far off as their own rounding, which
    is evenly spread below half a step: 0.29 steps of 2 U relative to the value's power of two, 0.42 U of the value on average (0.58 at worst)."""
    import torch

    h, w, t, _, _ = _inputs(rows, 256, 3000, getattr(torch, dtype))
    n = bs.head_loss(h, w, t)["log_norms"]
    one = torch.full((rows,), 1.0 / rows, device="cuda")
    b = bs.head_loss_backward(h, w, t, n, one)
    gh, _, gw, _ = O.Loss(h, w, t).grads(one)
    for got, want in ((b["grad_hidden"], gh), (b["grad_weight"], gw)):
        assert ((got.double() - want).norm() / want.norm()).item() <= 0.58 * O.U[h.dtype]


def test_strided_and_unaligned_rows(bs):
    import torch

    h, w, t, dl, _ = _inputs(70, 136, 900, torch.bfloat16)
    wide = torch.full((70, 151), float("nan"), dtype=h.dtype, device="cuda")
    weight = torch.full((900, 160), float("nan"), dtype=h.dtype, device="cuda")
    weight[:, 8:144] = w
    ref = bs.head_loss(h, w, t)
    for shift in (0, 1, 8):
        view = wide[:, shift:shift + 136]
        view.copy_(h)
        f = bs.head_loss(view, weight[:, 8:144], t)
        assert torch.equal(f["loss"], ref["loss"]) and torch.equal(f["log_norms"], ref["log_norms"])
        _check(bs, view, weight[:, 8:144], t, dl)


def test_rows_without_a_loss_may_hold_anything(bs):
    import torch

    h, w, t, dl, dn = _inputs(200, 128, 1500, torch.bfloat16, ignored=0.4)
    f, b = _check(bs, h, w, t, dl, dn)
    off = t < 0
    h2, dl2, dn2 = h.clone(), dl.clone(), dn.clone()
    h2[off] = float("nan")
    h2[off.nonzero()[::2, 0]] = float("inf")
    dl2[off], dn2[off] = float("inf"), float("nan")
    f2 = bs.head_loss(h2, w, t)
    assert torch.equal(f2["loss"], f["loss"]) and torch.equal(f2["log_norms"], f["log_norms"])
    b2 = bs.head_loss_backward(h2, w, t, f2["log_norms"], dl2, grad_log_norms=dn2)
    assert torch.equal(b2["grad_hidden"], b["grad_hidden"]) and torch.equal(b2["grad_weight"], b["grad_weight"])


@pytest.mark.parametrize("rows", [1, 130, 1030])
def test_no_row_has_a_loss(bs, rows):
    import torch

    h, w, t, dl, _ = _inputs(rows, 64, 700, torch.float16)
    h[:] = float("nan")
    f = bs.head_loss(h, w, torch.full_like(t, -1))
    b = bs.head_loss_backward(h, w, torch.full_like(t, -1), f["log_norms"], dl)
    for x in (*f.values(), *b.values()):
        assert (x == 0).all()


def test_no_rows(bs):
    import torch

    h, w, t, dl, _ = _inputs(4, 64, 700, torch.float16)
    f = bs.head_loss(h[:0], w, t[:0])
    assert f["loss"].shape == (0,)
    b = bs.head_loss_backward(h[:0], w, t[:0], f["log_norms"], dl[:0])
    assert b["grad_hidden"].shape == (0, 64) and (b["grad_weight"] == 0).all()


def test_targets_outside_the_vocabulary(bs):
    import torch

    h, w, t, dl, _ = _inputs(150, 64, 700, torch.bfloat16)
    t[3], t[149] = 700, 2 ** 31 - 1
    f = bs.head_loss(h, w, t)
    bad = torch.tensor([3, 149], device="cuda")
    assert torch.isnan(f["loss"][bad]).all() and torch.isnan(f["log_norms"][bad]).all()
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl)
    assert (b["grad_hidden"][bad] == 0).all()
    t2 = t.clone()
    t2[bad] = -1
    f2 = bs.head_loss(h, w, t2)
    b2 = bs.head_loss_backward(h, w, t2, f2["log_norms"], dl)
    ok = t2 >= 0
    assert torch.equal(f["loss"][ok], f2["loss"][ok]) and torch.equal(b["grad_weight"], b2["grad_weight"]) and torch.equal(b["grad_hidden"], b2["grad_hidden"])


def test_one_gradient_at_a_time(bs):
    import torch

    h, w, t, dl, _ = _inputs(140, 200, 30_000, torch.bfloat16)
    n = bs.head_loss(h, w, t)["log_norms"]
    both = bs.head_loss_backward(h, w, t, n, dl)
    one = bs.head_loss_backward(h, w, t, n, dl, want_weight=False)
    two = bs.head_loss_backward(h, w, t, n, dl, want_hidden=False)
    assert list(one) == ["grad_hidden"] and list(two) == ["grad_weight"]
    assert torch.equal(one["grad_hidden"], both["grad_hidden"]) and torch.equal(two["grad_weight"], both["grad_weight"])


@pytest.mark.parametrize("factor", [0.0, 2.0 ** -60, 2.0 ** -13, 4096.0])
def test_factors_of_any_size(bs, factor):
    """The gradients of the logits are rounded relative to their largest factor: powers of two change nothing."""
    import torch

    h, w, t, dl, _ = _inputs(140, 200, 3000, torch.bfloat16)
    n = bs.head_loss(h, w, t)["log_norms"]
    ref = bs.head_loss_backward(h, w, t, n, dl)
    got = bs.head_loss_backward(h, w, t, n, dl * factor)
    for k in ref:
        assert torch.equal(got[k].double(), ref[k].double() * factor), k


def test_large_logits(bs):
    """Logits beyond +-10,000: the largest alone counts, nothing overflows."""
    import torch

    h, w, t, dl, _ = _inputs(20, 64, 3000, torch.float16, std=1000.0)
    h = h.clamp(-100, 100)
    _check(bs, h, w, t, dl)


def test_what_is_not_finite_stays_in_its_row(bs):
    import torch

    h, w, t, dl, _ = _inputs(135, 64, 3000, torch.bfloat16)
    ref = bs.head_loss(h, w, t)
    h[7, 3], h[131, 5] = float("nan"), float("inf")
    f = bs.head_loss(h, w, t)
    bad = torch.zeros(135, dtype=torch.bool, device="cuda")
    bad[[7, 131]] = True
    assert torch.isnan(f["loss"][bad]).all()
    assert torch.equal(f["loss"][~bad], ref["loss"][~bad])
    clean = bs.head_loss_backward(h, w, t, ref["log_norms"], dl, want_weight=False)["grad_hidden"]
    assert torch.isnan(clean[bad]).any(1).all() and torch.isfinite(clean[~bad]).all()


def test_gradients_against_differences(bs):
    """Central differences of the kernel's own losses along a direction that the 16 bits hold exactly.  The third
    derivative of a loss along it is at most 2 * spread^3 of the logits' derivative, so the quotient is off by e^2 / 3 * spread^3, and by the
    losses' errors over e."""
    import torch

    rows, width, vocab, e = 6, 64, 300, 2.0 ** -5
    g = torch.Generator(device="cuda").manual_seed(5)
    h = torch.randint(-64, 65, (rows, width), generator=g, device="cuda").float() / 64
    d = torch.randint(-1, 2, (rows, width), generator=g, device="cuda").float()
    w = (torch.randn((vocab, width), generator=g, device="cuda") * 0.1).to(torch.float16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    one = torch.ones(rows, device="cuda")
    f = [bs.head_loss((h + k * e * d).half(), w, t) for k in (-1, 0, 1)]
    want = [O.Loss((h + k * e * d).half(), w, t) for k in (-1, 1)]
    gh = bs.head_loss_backward(h.half(), w, t, f[1]["log_norms"], one, want_weight=False)["grad_hidden"]
    _, dh, _, _ = O.Loss(h.half(), w, t).grads(one)
    slope = d.double() @ w.double().T
    spread = slope.amax(1) - slope.amin(1)
    quotient = (f[2]["loss"].double() - f[0]["loss"].double()) / (2 * e)
    bound = e * e / 3 * spread ** 3 + (want[0].d_loss + want[1].d_loss) / (2 * e) + (dh * d.abs().double()).sum(1)
    _near("difference", (gh.double() * d.double()).sum(1), quotient, bound)


@pytest.mark.parametrize("cap", [1e-40, 1e-6, 1e30])
def test_soft_caps_of_any_size(bs, cap):
    """A cap of almost nothing leaves equal logits, a large one leaves them as they are."""
    import torch

    h, w, t, dl, _ = _inputs(40, 64, 900, torch.bfloat16)
    h[3] = 0
    f = bs.head_loss(h, w, t, softcap=cap)
    if cap < 1:
        assert ((f["log_norms"].double() - math.log(900)).abs() <= 2 * cap + 2e-6).all() and ((f["loss"].double() - math.log(900)).abs() <= 4 * cap + 2e-6).all()
    else:
        want = O.Loss(h, w, t)  # tanh's own error is 2^-22 of the cap: nothing is left of the logits
        assert torch.isfinite(f["loss"]).all() and (f["loss"].double() - want.loss).abs().max() <= cap


def test_repeats_are_equal(bs):
    import torch

    h, w, t, dl, _ = _inputs(400, 512, 30_000, torch.bfloat16, ignored=0.2)
    f = bs.head_loss(h, w, t)
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl)
    for _ in range(3):
        f2 = bs.head_loss(h, w, t)
        b2 = bs.head_loss_backward(h, w, t, f["log_norms"], dl)
        assert all(torch.equal(f[k], f2[k]) for k in f) and all(torch.equal(b[k], b2[k]) for k in b)


def test_streams_beside_one_another(bs):
    """Two calls at once, each on a stream of its own, of one handle."""
    import torch

    sets = [_inputs(300, 256, 20_000, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [(f := bs.head_loss(h, w, t), bs.head_loss_backward(h, w, t, f["log_norms"], dl)) for h, w, t, dl, _ in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (h, w, t, dl, _) in enumerate(sets):
            raw = streams[i] if i else streams[i].cuda_stream
            f = bs.head_loss(h, w, t, stream=raw)
            got[i].append((f, bs.head_loss_backward(h, w, t, f["log_norms"], dl, stream=raw)))
    torch.cuda.synchronize()
    for i in range(2):
        for f, b in got[i]:
            assert all(torch.equal(f[k], want[i][0][k]) for k in f) and all(torch.equal(b[k], want[i][1][k]) for k in b)


def test_captured_steps(bs):
    """Two graphs of a training step, replayed beside one another on new inputs."""
    import torch

    sets = [_inputs(200, 128, 9000, torch.float16, seed=s, ignored=0.2) for s in (1, 2, 3, 4)]
    steps = []
    for h, w, t, dl, _ in sets[:2]:
        args = [x.clone() for x in (h, w, t, dl)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f = bs.head_loss(*args[:3])
            bs.head_loss_backward(*args[:3], f["log_norms"], args[3])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            f = bs.head_loss(*args[:3])
            b = bs.head_loss_backward(*args[:3], f["log_norms"], args[3])
        steps.append((graph, side, args, f, b))
    for (graph, side, args, f, b), (h, w, t, dl, _) in zip(steps, sets[2:]):
        for x, y in zip(args, (h, w, t, dl)):
            x.copy_(y)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, side, *_ in steps:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for (graph, side, args, f, b), (h, w, t, dl, _) in zip(steps, sets[2:]):
        f2 = bs.head_loss(h, w, t)
        b2 = bs.head_loss_backward(h, w, t, f2["log_norms"], dl)
        assert all(torch.equal(f[k], f2[k]) for k in f) and all(torch.equal(b[k], b2[k]) for k in b)


def test_outputs_are_written_again_and_nothing_else(bs):
    import torch

    h, w, t, dl, _ = _inputs(33, 72, 777, torch.bfloat16)
    f = bs.head_loss(h, w, t)
    b = bs.head_loss_backward(h, w, t, f["log_norms"], dl)
    room = torch.full((4, 40), 7.0, device="cuda")
    out = {"loss": room[1, :33], "log_norms": room[2, :33]}
    assert bs.head_loss(h, w, t, out=out) is out
    assert torch.equal(out["loss"], f["loss"]) and (room[[0, 3]] == 7).all() and (room[:, 33:] == 7).all()
    room_h, room_w = torch.full((35, 72), 7.0, dtype=h.dtype, device="cuda"), torch.full((779, 72), 7.0, dtype=h.dtype, device="cuda")
    grads = {"grad_hidden": room_h[1:34], "grad_weight": room_w[1:778]}
    bs.head_loss_backward(h, w, t, f["log_norms"], dl, out=grads)
    assert torch.equal(grads["grad_hidden"], b["grad_hidden"]) and torch.equal(grads["grad_weight"], b["grad_weight"])
    assert (room_h[[0, 34]] == 7).all() and (room_w[[0, 778]] == 7).all()


def test_refusals(bs):
    import torch
    from opentail.stingray_b200 import StingrayError

    h, w, t, dl, _ = _inputs(8, 64, 100, torch.bfloat16)
    n = torch.zeros(8, device="cuda")
    for bad in (dict(hidden=h.half()), dict(hidden=h[:, :56]), dict(weight=w.float()), dict(weight=w.T), dict(targets=t.long()), dict(targets=t[:7]),
                dict(hidden=h.cpu()), dict(hidden=h[0])):
        a = {"hidden": h, "weight": w, "targets": t, **bad}
        with pytest.raises(ValueError):
            bs.head_loss(**a)
        with pytest.raises(ValueError):
            bs.head_loss_backward(**a, log_norms=n, grad_loss=dl)
    for bad in (dict(log_norms=n.double()), dict(grad_loss=dl[:3]), dict(grad_log_norms=n.cpu())):
        with pytest.raises(ValueError):
            bs.head_loss_backward(**{"hidden": h, "weight": w, "targets": t, "log_norms": n, "grad_loss": dl, **bad})
    odd = torch.zeros((100, 60), dtype=torch.bfloat16, device="cuda")
    for a, code in ((dict(hidden=h[:, :60], weight=odd), 4), (dict(softcap=-1.0), 1), (dict(softcap=float("nan")), 1), (dict(softcap=float("inf")), 1),
                    (dict(hidden=h[:, :56], weight=w[:, 1:57]), 4), (dict(hidden=h[:, :56], weight=torch.zeros((100, 60), dtype=h.dtype, device="cuda")[:, :56]), 4)):
        with pytest.raises(StingrayError) as e:
            bs.head_loss(**{"hidden": h, "weight": w, "targets": t, **a})
        assert e.value.code == code, a
    with pytest.raises(StingrayError):
        bs.head_loss_backward(h, w, t, n, dl, want_hidden=False, want_weight=False)
    assert np.isfinite(bs.head_loss(h, w, t)["loss"].cpu().numpy()).all()  # the handle goes on
