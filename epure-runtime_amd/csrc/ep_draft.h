// Descriptor and launcher of the verification of drafted tokens (draft.hip).
// Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ep {

// Strides in elements: b of sequences, s of steps; values of the vocabulary are adjacent.
struct DraftTensors {
    const void *target, *draft;      // [B][n + 1][V], [B][n][V] or NULL
    int64_t p_sb, p_ss, q_sb, q_ss;
    const int64_t *drafted;          // [B][n]
    int64_t d_sb, d_ss;
    const float *uniforms;           // [B][n + 1]
    int64_t u_sb, u_ss;
    int64_t V;
    int n;
};

size_t verify_workspace(int64_t B, int64_t V);
int launch_verify(const DraftTensors &t, int64_t B, int dtype, int64_t *accepted, int64_t *tokens, void *ws,
                  size_t ws_bytes, hipStream_t stream);

}  // namespace ep
