// Linear attention's launches, shared by the token-by-token kernel and its entry
// points (linear.hip) and the kernels that go by chunks (linear_chunk_kernels.hpp).
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

// Calls by chunks of tokens.  A whole chunk keeps its factors in the entry of its first
// row over kChunk, a request's last and shorter one in entry n_tokens / kChunk + s:
// whole chunks of other requests begin at least kChunk rows away, so requests that share
// no row share no entry, in whatever order they lie.
constexpr uint32_t kChunk = 64;
constexpr uint32_t kPrepThreads = 256;
constexpr uint32_t kXcds = 8;

struct ChunkPlan {
    bool chunked = false;
    uint32_t entries = 0;
    uint32_t chunks = 0;    // most of one request
    uint64_t key_bytes = 0, head_bytes = 0;  // of an entry, per key head and per head
    uint32_t segs = 1, seg_chunks = 0;       // segments of a request, at most, and their chunks
    uint64_t seg_decays = 0, seg_states = 0;  // where they are in the workspace
    uint64_t bytes = 0;
};

constexpr uint32_t kFragBytes = 1024;  // a 16 x 32 operand of f16: 16 bytes a lane
constexpr uint32_t kLowerFrags = 5;    // of a 64 x 64 lower triangle (lower_frag)
constexpr uint32_t kHeadBytes = 1024;  // a head's entry begins with ChunkHead

struct ChunkParams {
    LinearParams a;
    uint8_t *keys;   // [entries][key heads]: fragments of K, Q, K^T
    uint8_t *heads;  // [entries][heads]: ChunkHead, fragments of T (delta), P (outs)
    uint64_t key_bytes, head_bytes;
    uint32_t chunks;
    int type;
    uint32_t dim_k;
    uint32_t delta, outs;
    uint32_t segs, seg_chunks, second_pass;
    float *seg_states;  // [requests][segs][heads][Dk][Dv]
    float *seg_decays;  // [requests][segs][heads]
};

// The launches of a call by chunks, each only where the one before was made (prepare and
// walk; in segments also the scan and a second walk), and the loading of their code
// object, for rows of each type.
void launch_linear_chunks_f32(hipStream_t stream, const ChunkParams &p);
void launch_linear_chunks_f16(hipStream_t stream, const ChunkParams &p);
void launch_linear_chunks_bf16(hipStream_t stream, const ChunkParams &p);
bool load_linear_chunks_f32();
bool load_linear_chunks_f16();
bool load_linear_chunks_bf16();

}  // namespace kvmem_hip
