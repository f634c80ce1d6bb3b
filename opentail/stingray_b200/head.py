"""A head's weight in 4 bits, laid out for ``BatchSampler.head_logits`` (``PackedHead``).  Nothing is computed here;
``BatchSampler.head_*`` hands it to the library.

    head = bs.head_pack(codes, scales, zeros)             # once, when the model is loaded
    logits = bs.head_logits(hidden, head)                 # [rows, vocab] of a decode step
    tokens = bs.sample_rows(logits, params, uniforms=u)["tokens"]
"""
from __future__ import annotations


class PackedHead:
    """What ``BatchSampler.head_pack`` returns: a weight ``[vocab, width]`` in 4 bits with a scale, and a zero point where
    ``has_zeros``, per ``group`` columns.  ``packed`` is the device memory it lies in."""

    def __init__(self, packed, vocab: int, width: int, group: int, scale_dtype: int, has_zeros: bool):
        self.packed, self.vocab, self.width, self.group = packed, vocab, width, group
        self.scale_dtype, self.has_zeros, self.device_index = scale_dtype, has_zeros, packed.get_device()

    @property
    def nbytes(self) -> int:
        return self.packed.numel()
