// Linear attention's launches, shared by the token-by-token kernel and its entry
// points (linear.hip) and the kernels that go by chunks (linear_chunk.hip).
#pragma once

#include "recurrent.hpp"

namespace kvmem_hip {

struct LinearParams {
    BatchArgs batch;
    const uint8_t *q, *k, *v;
    uint64_t q_nb1, q_nb2, k_nb1, k_nb2, v_nb1, v_nb2;
    const uint8_t *decay, *beta;
    uint64_t decay_nb, beta_nb;
    const float *state;
    float *state_out;
    uint8_t *out;
    int out_type;
    uint32_t n_seq;
    uint32_t n_head;
    uint32_t group;   // heads of one key head
    uint32_t dim_v;
    uint32_t slices;  // of dim_v
    float scale;
};

// Calls by chunks of tokens.  Request s's chunk c keeps its factors in entry
// q_start[s] / kChunk + s + c: entries of ascending requests never meet.
constexpr uint32_t kChunk = 64;
constexpr uint32_t kPrepThreads = 256;

constexpr uint32_t kChunkFrom = 24;  // tokens a request from which a call goes by chunks

struct ChunkPlan {
    bool chunked = false;
    int p_parts = 0;        // f16 parts of the scores (0: no out)
    uint32_t entries = 0;
    uint32_t chunks = 0;    // most of one request
    uint32_t cols = 0;      // of dim_v per wave
    uint64_t key_bytes = 0, head_bytes = 0;  // of an entry, per key head and per head
    uint64_t bytes = 0;
};

bool load_linear_chunk_kernels();
ChunkPlan plan_chunks(const kvmem_hip_linear_args *a, uint32_t max_q);
// Both launches of a call by chunks (the second only where the first was made).
void launch_linear_chunks(hipStream_t stream, int type, uint32_t dim_k, const ChunkPlan &pl, const LinearParams &p,
                          uint8_t *workspace);

}  // namespace kvmem_hip
