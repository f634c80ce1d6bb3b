"""Head calls on another stream than the current one: results, workspaces and arguments whose tensors are dropped while the stream is still busy.
What torch's allocator hands out in between must be nobody else's memory.  Each busy stream sleeps for some 50 ms."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
SLEEP = 100_000_000  # cycles


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=4, max_vocab=64, max_history=1, max_top_k=1)
    yield b
    b.close()


@pytest.fixture(scope="module")
def data(bs):
    """Inputs of all calls, whose results are a few sizes: [1000] float32, [1000, 64], [900, 64] and [1000, 900] of them."""
    g = torch.Generator(device="cuda").manual_seed(1)
    w = (torch.randn((900, 64), generator=g, device="cuda") / 8).to(torch.bfloat16)
    h = torch.randn((1000, 64), generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, 900, (1000,), generator=g, device="cuda", dtype=torch.int32)
    dl = torch.rand(1000, generator=g, device="cuda")
    c = torch.randint(0, 256, (900, 32), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand((900, 2), generator=g, device="cuda") / 8).to(torch.float16)
    n = bs.head_loss(h, w, t)["log_norms"]
    head = bs.head_pack(c, s)
    torch.cuda.synchronize()
    return dict(h=h, w=w, t=t, dl=dl, n=n, c=c, s=s, head=head)


def _call(bs, d, kind, stream):
    """The tensors that a call writes."""
    if kind == "loss":
        return bs.head_loss(d["h"], d["w"], d["t"], stream=stream)
    if kind == "backward":
        return bs.head_loss_backward(d["h"], d["w"], d["t"], d["n"], d["dl"], stream=stream)
    if kind == "pack":
        return {"packed": bs.head_pack(d["c"], d["s"], stream=stream).packed}
    return {"logits": bs.head_logits(d["h"], d["head"], stream=stream)}


KINDS = ["loss", "backward", "pack", "logits"]


def _streams():
    s = torch.cuda.Stream()
    return {"torch's": s, "a handle": s.cuda_stream}


@pytest.mark.parametrize("which", ["torch's", "a handle"])
@pytest.mark.parametrize("kind", KINDS)
def test_dropped_results_are_not_handed_out_again(bs, data, kind, which):
    stream = _streams()[which]
    shapes = {k: (tuple(x.shape), x.dtype) for k, x in _call(bs, data, kind, None).items()}
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(getattr(stream, "cuda_stream", stream))):
        torch.cuda._sleep(SLEEP)
    _call(bs, data, kind, stream)
    fresh = [torch.full(shape, 7, dtype=dtype, device="cuda") for shape, dtype in shapes.values() for _ in range(4)]
    torch.cuda.synchronize()
    assert all((x == 7).all() for x in fresh)


@pytest.mark.parametrize("which", ["torch's", "a handle"])
@pytest.mark.parametrize("kind", KINDS)
def test_what_the_current_stream_still_reads_is_not_written(bs, data, kind, which):
    stream = _streams()[which]
    old = {k: torch.full_like(x, 3) for k, x in _call(bs, data, kind, None).items()}
    copies = {k: torch.empty_like(x) for k, x in old.items()}
    torch.cuda.synchronize()
    torch.cuda._sleep(SLEEP)
    for k in copies:
        copies[k].copy_(old.pop(k))
    _call(bs, data, kind, stream)
    torch.cuda.synchronize()
    assert all((x == 3).all() for x in copies.values())


@pytest.mark.parametrize("which", ["torch's", "a handle"])
@pytest.mark.parametrize("kind", KINDS)
def test_results_that_the_current_stream_reads_last(bs, data, kind, which):
    """Waited for, read on the current stream and dropped: the next call on the other stream does not write into them."""
    stream = _streams()[which]
    want = _call(bs, data, kind, None)
    torch.cuda.synchronize()
    other = {**data, "h": -data["h"], "c": ~data["c"]}
    copies = []
    for _ in range(3):
        got = _call(bs, data, kind, stream)
        torch.cuda.synchronize()
        torch.cuda._sleep(SLEEP)
        copies.append({k: torch.empty_like(x).copy_(x) for k, x in got.items()})
        del got
        _call(bs, other, kind, stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x[k], want[k]) for x in copies for k in want)


@pytest.mark.parametrize("kind", KINDS)
def test_arguments_dropped_at_once(bs, data, kind):
    stream = torch.cuda.Stream()
    want = _call(bs, data, kind, None)
    torch.cuda.synchronize()
    copies = {k: x.clone() for k, x in data.items() if k != "head"}
    copies["head"] = bs.head_pack(copies["c"], copies["s"])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(SLEEP)
    got = _call(bs, copies, kind, stream)
    del copies
    fresh = [torch.full_like(x, 1) for k, x in data.items() if k != "head" for _ in range(3)]
    fresh += [torch.full_like(data["head"].packed, 0x77) for _ in range(3)]
    torch.cuda.synchronize()
    assert len(fresh) > 3 and all(torch.equal(got[k], want[k]) for k in want)


def test_the_default_stream_by_its_handle(bs, data):
    """Handle 0 is the default stream, not some stream of the pool; the current stream's own handle is no other stream."""
    want = bs.head_loss(data["h"], data["w"], data["t"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    assert torch.cuda.default_stream().cuda_stream == 0 and bs._aside(0) is None
    with torch.cuda.stream(side):
        assert bs._aside(0).cuda_stream == 0 and bs._aside(side.cuda_stream) is None and bs._aside(side) is None
        got = bs.head_loss(data["h"], data["w"], data["t"], stream=0)
    torch.cuda.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
    assert math.isfinite(got["loss"].sum().item())


@pytest.mark.parametrize("kind", KINDS)
def test_a_stream_forked_inside_a_capture(bs, data, kind):
    """The call's stream joins a capture on another one; its results and workspace are the graph's."""
    want = _call(bs, data, kind, None)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        got = _call(bs, data, kind, side)
        torch.cuda.current_stream().wait_stream(side)
        copies = {k: x.clone() for k, x in got.items()}
    for x in [*got.values(), *copies.values()]:
        x.zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(got[k], want[k]) and torch.equal(copies[k], want[k]) for k in want)
