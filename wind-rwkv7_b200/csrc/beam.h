// Interface between the C ABI (capi.cu) and beam search's kernels (beam.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace wkv7 {

constexpr int BEAM_MAX_K = 64, BEAM_MAX_W = 64;

struct BeamParams {
    const void* logits;             // [B, W, V], strides (sb, sw, 1)
    const float* scores;            // [B, W]
    const unsigned char* finished;  // [B, W] or null
    float* out_scores;              // [B, k]
    int64_t *parents, *tokens;      // [B, k]
    unsigned char* out_finished;    // [B, k], with finished
    float *seg_max, *part;          // workspace: [B, W, segments], [B, W, parts, 2]
    long long sb, sw;
    int B, W, V, k, eos, segments, parts, per_part;
    bool f32;
};
size_t beam_workspace_bytes(long long B, long long W, long long V);
int launch_beam_select(BeamParams p, void* workspace, cudaStream_t stream);

constexpr int REORDER_MAX = 64;  // tensors of one launch
struct ReorderParams {
    const void* src[REORDER_MAX];
    void* dst[REORDER_MAX];
    long long row_bytes[REORDER_MAX], src_pitch[REORDER_MAX], dst_pitch[REORDER_MAX];
    const void* parents;  // [B, k]
    int B, W, k, count;
    bool idx64, keep;     // keep: a row whose parent does not exist is src's own, not zero
    int* status;
};
int launch_reorder(const ReorderParams& p, cudaStream_t stream);

}  // namespace wkv7
