"""Calls on another stream than the current one allocate their results there: one dropped at once is not handed out again while the stream is
busy, nor is memory written that the current stream still reads.  Each busy stream sleeps for some 50 ms."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
SLEEP = 100_000_000  # cycles
ROWS, VOCAB = 8, 1000


@pytest.fixture(scope="module")
def bs():
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler(max_rows=ROWS, max_vocab=VOCAB, max_history=8, max_top_k=64, max_spec_draft=3, max_cached_masks=4)
    b.mask_cache_put(1, np.full((VOCAB + 31) // 32, 0x55555555, np.uint32), VOCAB)
    torch.cuda.synchronize()
    yield b
    b.close()


@pytest.fixture(scope="module")
def data():
    from opentail.stingray_b200 import SamplingParams

    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn((ROWS, VOCAB), generator=g, device="cuda")
    u = np.linspace(0.05, 0.95, ROWS).astype(np.float32)
    p = torch.softmax(logits, 1)
    q = torch.softmax(torch.randn((ROWS, VOCAB), generator=g, device="cuda"), 1)
    draft = torch.randint(0, VOCAB, (2, 3), generator=g, device="cuda", dtype=torch.int32)
    trail = torch.zeros((4, 2, 4), dtype=torch.int32, device="cuda")
    # (everything is there before a call: what it is given has to be ready on its stream)
    return dict(draft_logits=q[:6].reshape(2, 3, VOCAB).log(), tokens=draft.flatten().repeat(2)[:ROWS].contiguous(), scores=torch.zeros((2, 4), device="cuda"), logits=logits, u=u, p=p, q=q, draft=draft, trail=trail, params=[SamplingParams(TopK=40)] * ROWS, full=[SamplingParams(TopK=0, TopP=0.9)] * ROWS,
                masks=torch.full((2, ROWS, (VOCAB + 31) // 32), 0x0F0F0F0F, dtype=torch.int32, device="cuda"), zero=torch.zeros((2, 4), dtype=torch.int32, device="cuda"))


def _call(bs, d, kind, stream):
    """The tensors that a call writes, by their places among its results."""
    lg = d["logits"]
    if kind == "sample_rows":
        r = bs.sample_rows(lg, d["params"], uniforms=d["u"], want_probs=True, want_flags=True, want_topk=40, stream=stream)
    elif kind == "argmax_rows":
        r = bs.argmax_rows(lg, stream=stream)
    elif kind == "build_distribution":
        r = [bs.build_distribution(lg, d["full"], stream=stream)]
    elif kind == "sample_with_distribution":
        r = bs.sample_with_distribution(lg, d["full"], uniforms=d["u"], stream=stream)
    elif kind == "sample_from_probs":
        r = bs.sample_from_probs(d["p"], d["u"], stream=stream)
    elif kind == "resample_residual":
        r = bs.resample_residual(d["p"], d["q"], np.stack([d["u"], d["u"]], 1), stream=stream)
    elif kind == "spec_verify":
        r = bs.spec_verify(lg.view(2, 4, VOCAB), d["draft_logits"], d["draft"], d["params"][:2], np.full((2, 5), 0.4), want_probs=True, stream=stream)
    elif kind == "mtp_accept":
        r = bs.mtp_accept(lg, d["tokens"], 0.5, stream=stream)
    elif kind == "and_masks":
        r = bs.and_masks(d["masks"], VOCAB, stream=stream)
    elif kind == "mask_compose":
        r = bs.mask_compose(np.full((ROWS, 1), 1), VOCAB, stream=stream)
    elif kind == "beam_select":
        r = bs.beam_select(lg, d["scores"], want_norms=True, want_flags=True, stream=stream)
    else:
        r = bs.beam_backtrace(d["trail"], d["trail"], d["zero"], d["zero"], d["zero"], stream=stream)
    return dict(r.items() if isinstance(r, dict) else enumerate(r))


KINDS = ["sample_rows", "argmax_rows", "build_distribution", "sample_with_distribution", "sample_from_probs", "resample_residual", "spec_verify", "mtp_accept", "and_masks",
         "mask_compose", "beam_select", "beam_backtrace"]


@pytest.mark.parametrize("kind", KINDS)
def test_dropped_results_are_not_handed_out_again(bs, data, kind):
    shapes = [(tuple(x.shape), x.dtype) for x in _call(bs, data, kind, None).values()]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(SLEEP)
    _call(bs, data, kind, stream)
    fresh = [torch.full(shape, 7, dtype=dtype, device="cuda") for shape, dtype in shapes for _ in range(4)]
    torch.cuda.synchronize()
    assert all((x == 7).all() for x in fresh)


@pytest.mark.parametrize("kind", KINDS)
def test_results_are_right_and_leave_alone_what_the_current_stream_reads(bs, data, kind):
    want = {k: x.clone() for k, x in _call(bs, data, kind, None).items()}
    old = {k: torch.full_like(x, 3, memory_format=torch.contiguous_format) for k, x in want.items()}
    copies = {k: torch.empty_like(x) for k, x in old.items()}
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(SLEEP)
    for k in copies:
        copies[k].copy_(old.pop(k))
    got = _call(bs, data, kind, stream.cuda_stream)
    torch.cuda.synchronize()
    assert all((x == 3).all() for x in copies.values())
    assert all(torch.equal(got[k].view(torch.uint8) if got[k].dtype == torch.float32 and got[k].is_contiguous() else got[k],
                           want[k].view(torch.uint8) if got[k].dtype == torch.float32 and got[k].is_contiguous() else want[k]) for k in want)
