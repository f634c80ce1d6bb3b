"""What the beam calls decide on the host: the layout of per-beam state, checked by walking it as the kernel does, the
struct sizes, and refusals that need no device."""
import ctypes as C

import numpy as np
import pytest


def _native():
    from opentail.stingray_b200 import _native as N
    from opentail.stingray_b200 import build as B

    B.build()
    N.load()
    return N


def test_struct_layouts():
    N = _native()
    assert (C.sizeof(N.StgBeamBatch), C.sizeof(N.StgBeamSearch), C.sizeof(N.StgBeamState), C.sizeof(N.StgBeamReorder)) == (120, 136, 72, 48)


def test_null_handles_are_refused():
    N = _native()
    lib = N.load()
    assert lib.stg_beam_select(None, None, None) == 1
    assert lib.stg_beam_start(None, None, 0, 0, None) == 1
    assert lib.stg_beam_advance(None, None, 1, None, None, None, 0, None) == 1
    assert lib.stg_beam_reorder(None, None, None) == 1
    assert lib.stg_beam_backtrace(None, None, None, 0, 0, 1, 0, None, None, None, 0, None, 0, None, None) == 1


def _walk(s, row, positions):
    """Byte offsets of a row that a reordering moves, as the description says."""
    sizes, inner = list(s.size), s.inner_bytes
    if positions is not None and s.position_dim == 3:
        inner = min(inner, positions * s.position_bytes)
    if positions is not None and 0 <= s.position_dim < 3:
        sizes[s.position_dim] = min(sizes[s.position_dim], positions)
    i2, i1, i0, b = np.ogrid[:sizes[2], :sizes[1], :sizes[0], :inner]
    return np.sort((row * s.row_stride + i2 * s.stride[2] + i1 * s.stride[1] + i0 * s.stride[0] + b).ravel())


@pytest.mark.parametrize("positions", [None, 0, 1, 3, 100])
def test_descriptions_cover_a_row_and_nothing_else(positions):
    import torch
    from opentail.stingray_b200 import BeamStates

    cases = [
        (torch.zeros(6, 2, 5, 4, dtype=torch.bfloat16), 0, 2), (torch.zeros(6, 2, 4, 5), 0, 3), (torch.zeros(6, 5, 2, 4), 0, 1),
        (torch.zeros(3, 6, 2, 5, 4), 1, 3), (torch.zeros(2, 3, 6, 5, 2, dtype=torch.int8), 2, 3), (torch.zeros(6, 5, dtype=torch.int32), 0, 1),
        (torch.zeros(6), 0, None), (torch.zeros(5, 6), 1, 0), (torch.zeros(6, 9, 8)[:, :5, :6], 0, 1), (torch.zeros(6, 4, 9, 8)[:, :, :5, ::2], 0, 2),
        (torch.zeros(6, 1, 5), 0, 1), (torch.zeros(6, 5, 1, 3), 0, 1), (torch.zeros(6, 3, 5).transpose(1, 2), 0, 1), (torch.zeros(5, 3, 6).permute(2, 1, 0), 0, 2),
    ]
    for t, beam, pos in cases:
        s = BeamStates._describe(t, beam, pos)
        where = np.arange(int(np.prod(t.shape))).reshape(t.shape)
        strides = np.array(t.stride()) * t.element_size()
        for row in range(6):
            part = t.select(beam, row)
            index = np.indices(t.shape).reshape(t.dim(), -1)
            keep = index[beam] == row
            if pos is not None and positions is not None:
                keep &= index[pos] < positions
            first = (index[:, keep] * strides[:, None]).sum(0)
            want = np.sort((first[:, None] + np.arange(t.element_size())).ravel())
            assert np.array_equal(_walk(s, row, positions if pos is not None else None), want), (tuple(t.shape), t.stride(), pos, positions)


def test_descriptions_are_short():
    """A cache's runs are as long as its layout allows."""
    import torch
    from opentail.stingray_b200 import BeamStates

    s = BeamStates._describe(torch.zeros(4, 8, 64, 32, dtype=torch.bfloat16), 0, 2)
    assert (s.inner_bytes, s.position_bytes, s.position_dim, list(s.size)) == (64 * 32 * 2, 64, 3, [8, 1, 1])
    s = BeamStates._describe(torch.zeros(4, 8, 64, 32), 0, None)
    assert (s.inner_bytes, s.position_dim, list(s.size)) == (8 * 64 * 32 * 4, -1, [1, 1, 1])
    with pytest.raises(ValueError, match="more than three"):
        BeamStates._describe(torch.zeros(8, 4, 4, 4, 4, 4)[:, ::2, ::2, ::2, ::2, ::2], 0, None)


@pytest.mark.parametrize("beams,eos", [(32, 4), (32, 8), (16, 8), (26, 4), (22, 5)])
def test_searches_that_need_more_candidates_than_there_may_be_are_refused(beams, eos):
    """With fewer than num_beams * (1 + end tokens) of them, fewer beams than num_beams may go on."""
    from opentail.stingray_b200 import BeamSearch

    with pytest.raises(ValueError, match="candidates a sequence"):
        BeamSearch(1, beams, 4, eos=range(2, 2 + eos))


@pytest.mark.parametrize("beams,eos", [(32, [5, 6, 7]), (25, [5, 6, 7, 8]), (32, [5] * 8), (14, list(range(8))), (32, [])])
def test_searches_of_as_many_candidates_as_there_may_be_are_not(beams, eos):
    import torch
    from opentail.stingray_b200 import BeamSearch

    if torch.cuda.is_available():
        assert BeamSearch(1, beams, 4, eos=eos).n_candidates == beams * (1 + len(set(eos)))
    else:  # refused for its device alone
        with pytest.raises(ValueError, match="CUDA device"):
            BeamSearch(1, beams, 4, eos=eos, device="cpu")


def test_dimensions_that_are_not_there_are_refused():
    import torch
    from opentail.stingray_b200 import BeamStates

    t = torch.zeros(8, 2, 5, 4)
    for kw in ({"beam_dim": 4}, {"beam_dim": -5}, {"position_dim": 4}, {"position_dim": 6}, {"position_dim": -5}, {"position_dim": [7]}):
        with pytest.raises(ValueError, match="no dimension"):
            BeamStates([t], 4, **kw)
    with pytest.raises(ValueError, match="no dimension"):
        BeamStates([torch.zeros(())], 1)
    with pytest.raises(ValueError, match="no dimension"):
        BeamStates([t, torch.zeros(8, 3)], 4, position_dim=2)
    for beams in (0, -4):
        with pytest.raises(ValueError, match="num_beams"):
            BeamStates([t], beams)
    for kw in ({"beam_dim": -4, "position_dim": -2}, {"beam_dim": 0, "position_dim": 3}):
        with pytest.raises(ValueError, match="CUDA device"):  # nothing else is wrong with these
            BeamStates([t], 4, **kw)


def test_states_and_searches_want_a_cuda_device():
    import torch
    from opentail.stingray_b200 import BeamSearch, BeamStates

    with pytest.raises(ValueError):
        BeamStates([torch.zeros(8, 4)], 4)
    with pytest.raises(ValueError):
        BeamStates([], 4)
    with pytest.raises(ValueError):
        BeamSearch(1, 4, 4, device="cpu")
