// Beam search on the device: selection over beams and vocabulary, and the reordering of the beams'
// states (beam.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/stt_b200.h"
#include "kv8.h"

namespace stt {

constexpr int kMaxBeams = 32;
constexpr int kBeamThreads = 128;
// Logits of a thread in a tile of 8 or 16 KB, which needs twice the registers for 16-bit logits; CTAs of an
// SM; logits of a tile.
constexpr int beam_per_thread(int dtype) { return dtype == DT_F32 ? 16 : 32; }
constexpr int beam_ctas(int dtype) { return dtype == DT_F32 ? 8 : 7; }
constexpr int beam_tile(int dtype) { return kBeamThreads * beam_per_thread(dtype); }
constexpr int kBeamMaxChunks = 32;                            // CTAs of a row

struct BeamArgs {
    const void* logits;   // [batch * beams][vocab], rows row_stride elements apart
    int64_t row_stride;
    int32_t batch, beams, vocab;
    int32_t chunks, tiles_per_chunk;  // CTAs of a row, tiles of a CTA
    const float* scores;  // [batch][beams]
    const uint8_t* done;  // [batch][beams] or NULL
    int32_t eos;          // -1: none
    float* next_scores;
    int32_t *parents, *tokens;
    uint8_t* next_done;   // or NULL
    // workspace, indexed by row * chunks + chunk
    float* part_max;
    double* part_sum;
    uint64_t* part_keys;  // [kMaxBeams of the selector] best keys of the chunk, descending
    int32_t key_stride;
    uint32_t* tickets;    // [batch]
    int32_t* err;
};

struct ReorderArgs {
    uint8_t* states;
    int64_t row_stride;    // bytes; segment s of a row starts at (s / inner) * outer_stride + (s % inner) * segment_stride
    int64_t segment_stride, outer_stride;
    int32_t segments, inner;
    int32_t first_segment; // of the launch
    int64_t units, unit_bytes;
    int32_t groups, beams;
    const int32_t* rows;   // place of each row (row_stride apart), or NULL: its number
    const int32_t* parents;
    const int32_t* held;   // what each row holds, or NULL: `units` units
    int32_t per_unit;      // of which `per_unit` make one unit
};

// The selector's device, and whether it was made for such a call.
int beam_device(const stt_beam* beam);
bool beam_fits(const stt_beam* beam, int batch, int beams, int vocab);
// stt_beam_select_device that raises `err` (a device word; NULL: the selector's own).
int beam_select(stt_beam* beam, const stt_beam_step* step, int32_t* err, cudaStream_t st);
cudaError_t launch_beam_select(const BeamArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_reorder(const ReorderArgs& a, cudaStream_t st);

}  // namespace stt
