// ssla_linattn.cuh -- what the linear-attention kernels share.
#pragma once

#include <vector>

#include "ssla_ops.cuh"

namespace ssla {
namespace ops {

struct LinArgs {
    const void *q, *k, *v;
    void* out;
    const float* decay;
    float* state;
    long long q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head, decay_row, decay_head;
    int n_rows, heads, q_share, k_share, dk, dv, n_slots;
    float scale;
    int stream;                     // step: the states are too many for L2
};

struct Seq {
    int start, len, slot;
};

// The chunked form of whole sequences (ssla_linattn_chunk.cu): its workspace
// and its launches on the current device.
size_t chunk_workspace(const LinArgs& a, int dtype, const std::vector<Seq>& seqs);
int chunk_launch(const LinArgs& a, int dtype, const std::vector<Seq>& seqs, void* workspace, cudaStream_t st);

int chunk_status(unsigned* bits);

}  // namespace ops
}  // namespace ssla
