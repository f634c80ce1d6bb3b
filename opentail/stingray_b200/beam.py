"""What a program that decodes with beams keeps beside its ``BatchSampler``: the search's device arrays (``BeamSearch``)
and the description of its per-beam state (``BeamStates``).  Nothing is computed here; ``BatchSampler.beam_*``
hands both to the library.  The reference has no beam search.

    bs = BatchSampler(max_rows=n_seq * beams, max_vocab=vocab)
    search = BeamSearch(n_seq, beams, max_steps=256, eos=[2])
    states = BeamStates(key_value_caches, beams, position_dim=2)      # tensors [n_seq * beams, heads, room, width]
    bs.beam_start(search)
    best = None
    for step in range(256):
        logits = model(search.tokens, ...)                            # [n_seq * beams, vocab]
        best = bs.beam_select(logits, search.scores, search.n_candidates, out=best)
        bs.beam_advance(search, best)
        bs.beam_reorder(states, search.parents, positions=used)
    found = bs.beam_backtrace(search.trail_tokens, search.trail_parents, search.pool_steps, search.pool_parents, search.pool_tokens)

Nothing in the loop reads the device back, so it can be captured into a CUDA graph; ``search.done`` says when every
sequence has ended.
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

from . import _native as N


class BeamSearch:
    """The device arrays of a search over ``n_seq`` sequences of ``num_beams`` beams, with a trail of ``max_steps`` tokens.

    A hypothesis of L tokens competes with its score divided by ``L ** length_penalty``.  ``n_candidates`` is how
    many candidates ``beam_select`` has to find so that ``num_beams`` go on whatever ends; a search that needs more than
    there may be (128: 32 beams and four end tokens, 16 and eight) is refused.  Call
    ``BatchSampler.beam_start`` before the first step, also for single sequences that a new request takes over."""

    def __init__(self, n_seq: int, num_beams: int, max_steps: int, *, eos: Sequence[int] = (), pad: int = 0, length_penalty: float = 1.0,
                 early_stopping: bool = False, device=None):
        import torch

        eos = [int(e) for e in eos]
        if not 1 <= num_beams <= N.BEAM_MAX_BEAMS:
            raise ValueError(f"num_beams must be 1 to {N.BEAM_MAX_BEAMS}")
        if n_seq < 0 or max_steps < 1:
            raise ValueError("n_seq must be >= 0 and max_steps >= 1")
        if len(eos) > N.BEAM_MAX_EOS:
            raise ValueError(f"at most {N.BEAM_MAX_EOS} end tokens")
        self.n_candidates = num_beams * (1 + len(set(eos)))
        if self.n_candidates > N.BEAM_MAX_CANDIDATES:
            raise ValueError(f"{num_beams} beams and {len(set(eos))} end tokens need {self.n_candidates} candidates a sequence so that {num_beams} go on "
                             f"whatever ends, more than {N.BEAM_MAX_CANDIDATES}")
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError("a search lies on a CUDA device")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.n_seq, self.num_beams, self.max_steps = n_seq, num_beams, max_steps
        self.eos, self.pad, self.device_index = eos, pad, dev.index

        def ints(*shape):
            return torch.zeros(shape, dtype=torch.int32, device=dev)

        def floats(*shape):
            return torch.zeros(shape, dtype=torch.float32, device=dev)

        B, K = n_seq, num_beams
        self.tokens, self.parents, self.scores = ints(B, K), ints(B, K), floats(B, K)
        self.steps, self.done = ints(B), ints(B)
        self.pool_scores, self.pool_steps, self.pool_parents, self.pool_tokens = floats(B, K), ints(B, K), ints(B, K), ints(B, K)
        self.trail_tokens, self.trail_parents = ints(max_steps, B, K), ints(max_steps, B, K)
        self.norms = torch.arange(1, max_steps + 1, dtype=torch.float64).pow(float(length_penalty)).to(dev)
        self._eos = (C.c_int32 * max(1, len(eos)))(*eos)
        self.struct = N.StgBeamSearch(
            C.sizeof(N.StgBeamSearch), B, K, max_steps, len(eos), pad, 1 if early_stopping else 0, C.addressof(self._eos),
            *(t.data_ptr() for t in (self.norms, self.tokens, self.parents, self.scores, self.steps, self.done, self.pool_scores, self.pool_steps,
                                     self.pool_parents, self.pool_tokens, self.trail_tokens, self.trail_parents)))


class BeamStates:
    """Per-beam state of a program, described once: CUDA tensors with ``n_seq * num_beams`` rows along ``beam_dim``, of any
    type and strides.  ``position_dim``: the dimension along which the tensors fill up as a sequence grows, so
    that ``beam_reorder`` moves the positions in use only; one number for all tensors, or one per tensor (None: the
    tensor's rows are moved whole)."""

    def __init__(self, tensors, num_beams: int, *, beam_dim: int = 0, position_dim=None):
        self.tensors = list(tensors)
        dims = list(position_dim) if isinstance(position_dim, (list, tuple)) else [position_dim] * len(self.tensors)
        if len(dims) != len(self.tensors):
            raise ValueError("one position_dim per tensor")
        if not self.tensors:
            raise ValueError("no tensors")
        if num_beams < 1:
            raise ValueError("num_beams must be >= 1")
        for t, p in zip(self.tensors, dims):  # a dimension that is not there would be taken for another one below
            for name, d in (("beam_dim", beam_dim), ("position_dim", p)):
                if d is not None and not -t.dim() <= d < t.dim():
                    raise ValueError(f"{name} {d} is no dimension of a tensor of shape {tuple(t.shape)}")
        self.rows, self.device_index = None, self.tensors[0].get_device()
        described = []
        for t, p in zip(self.tensors, dims):
            if not t.is_cuda or t.get_device() != self.device_index:
                raise ValueError("the tensors must lie on one CUDA device")
            beam, pos = beam_dim % t.dim(), None if p is None else p % t.dim()
            if self.rows is None:
                self.rows = t.shape[beam]
            if t.shape[beam] != self.rows or self.rows % num_beams != 0:
                raise ValueError(f"{t.shape[beam]} rows: the tensors need the same multiple of {num_beams} rows")
            if pos == beam:
                raise ValueError("the positions cannot be the beams")
            described.append(self._describe(t, beam, pos))
        self._array = (N.StgBeamState * len(described))(*described)
        self.count, self.address = len(described), C.addressof(self._array)

    @staticmethod
    def _describe(t, beam: int, pos) -> N.StgBeamState:
        size = t.element_size()
        dims = sorted((t.stride(d) * size, t.shape[d], d == pos) for d in range(t.dim()) if d != beam and (t.shape[d] != 1 or d == pos))
        run, per, of_run, outer = size, 0, False, []
        for stride, n, is_pos in dims:  # from the innermost on
            if not outer and not of_run and stride == run:
                if is_pos:  # the run may be cut off within it: nothing further joins the run
                    per, of_run = run, True
                run *= n
            elif outer and not outer[-1][2] and not is_pos and stride == outer[-1][0] * outer[-1][1] and n * outer[-1][1] < 1 << 31:
                outer[-1] = (outer[-1][0], outer[-1][1] * n, False)
            else:
                outer.append((stride, n, is_pos))
        if len(outer) > 3:
            raise ValueError(f"a row of shape {tuple(t.shape)} with strides {tuple(t.stride())} has more than three dimensions beside its contiguous runs")
        where = 3 if of_run else next((i for i, o in enumerate(outer) if o[2]), -1)
        outer += [(0, 1, False)] * (3 - len(outer))
        return N.StgBeamState(t.data_ptr(), t.stride(beam) * size, run, per, (C.c_int64 * 3)(*(o[0] for o in outer)),
                              (C.c_int32 * 3)(*(o[1] for o in outer)), where)
