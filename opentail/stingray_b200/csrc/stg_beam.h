// Beam search (stg_beam_*.cu): limits and the workspace of the selection.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../../include/stingray_sampler.h"
#include "stg_beam_pieces.h"
#include "stg_handle.h"

namespace stg {

// What one CTA leaves of its piece of a row: the sum of exp(x) over its logits, relative to a BeamRef (stg_beam_select.cu).
struct BeamPart {
    double s;
    float c, logit;
};

struct BeamWs {
    BeamPart *parts;    // [rows, pieces]
    float *tops;        // [rows, groups]: the largest logit of each group of neighbours
    uint32_t *tickets;  // [n_seq]: CTAs of a sequence that have ended; zero between calls
};

inline size_t beam_ws_bytes(StgHandle h)
{
    return ((size_t)h->cfg.max_rows + kBeamExtraPieces) * sizeof(BeamPart) + (size_t)h->cfg.max_rows * ((size_t)h->cfg.max_vocab / 512 + 1) * 4 + 1024;
}

// device arrays are checked for their elements' alignment, which the host can see
inline bool misaligned(const void *p, size_t to) { return ((uintptr_t)p % to) != 0; }

// The handle's device for the time of a call; the caller's is current again behind it.
struct OnDevice {
    int before = -1;
    cudaError_t error;
    explicit OnDevice(int device)
    {
        error = cudaGetDevice(&before);
        if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
        if (before == device) before = -1;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

int beam_check_rows(StgHandle h, const char *who, int32_t n_seq, int32_t n_beams);

}  // namespace stg
