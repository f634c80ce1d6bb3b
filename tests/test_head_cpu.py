"""What the head's calls decide on the host: struct sizes, null handles, and refusals that need no device."""
import ctypes as C

import pytest


def _native():
    from opentail.stingray_b200 import _native as N
    from opentail.stingray_b200 import build as B

    B.build()
    N.load()
    return N


def test_struct_layouts():
    N = _native()
    assert (C.sizeof(N.StgHeadLoss), C.sizeof(N.StgHeadPack), C.sizeof(N.StgHeadLogits)) == (128, 72, 104)


def test_null_handles_are_refused():
    lib = _native().load()
    assert lib.stg_head_loss_workspace(None, None, 0, None) == 1
    assert lib.stg_head_loss(None, None, None) == 1
    assert lib.stg_head_loss_backward(None, None, None) == 1
    assert lib.stg_head_pack_bytes(None, 1, 32, 32, 0, None) == 1
    assert lib.stg_head_pack(None, None, None) == 1
    assert lib.stg_head_logits_workspace(None, None, None) == 1
    assert lib.stg_head_logits(None, None, None) == 1


def _sampler():
    """A ``BatchSampler`` without a handle: what it refuses, it refuses before the library is asked."""
    from opentail.stingray_b200 import BatchSampler

    b = BatchSampler.__new__(BatchSampler)
    b.device, b._head_sizes, b._lib = 0, {}, None
    return b


def test_tensors_that_are_not_on_the_device_are_refused():
    import torch
    from opentail.stingray_b200 import PackedHead

    b = _sampler()
    h, w, t = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    f = torch.zeros(4)
    with pytest.raises(ValueError, match="cuda:0"):
        b.head_loss(h, w, t)
    with pytest.raises(ValueError, match="cuda:0"):
        b.head_loss_backward(h, w, t, f, f)
    with pytest.raises(ValueError, match="cuda:0"):
        b.head_pack(torch.zeros(100, 32, dtype=torch.uint8), torch.ones(100, 1, dtype=torch.float16))
    with pytest.raises(ValueError, match="handle on cuda:0"):
        b.head_logits(h, PackedHead(torch.zeros(16, dtype=torch.uint8), 100, 64, 64, 2, False))


def test_types_and_shapes_are_refused():
    import torch

    b = _sampler()
    t = torch.zeros(4, dtype=torch.int32)
    for w in (torch.zeros(100, 64), torch.zeros(64, dtype=torch.bfloat16), torch.zeros(2, 100, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.int8)):
        with pytest.raises(ValueError, match="weight must be a matrix"):
            b.head_loss(torch.zeros(4, 64, dtype=torch.bfloat16), w, t)
    for c in (torch.zeros(100, 32, dtype=torch.int8), torch.zeros(100, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="codes must be a matrix"):
            b.head_pack(c, torch.ones(100, 1, dtype=torch.float16))
