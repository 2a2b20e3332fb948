// Attention calls whose launch HIP cannot hold: refused by the host checks, before
// any HIP call, so the program runs without a GPU.  A dispatch counts at most 2^32 - 1
// work items: 2^24 workgroups of 256 threads (few queries) and 2^23 of 512 (many) are
// the first that do not fit.  Linked with libkvmem_hip.so; the context is a bare
// struct (no stream, no device).
#include <cstdio>
#include <string>

#include "kvmem_internal.hpp"

static kvmem_hip_ctx ctx;
static int bad = 0;

static void refused(const char *what, const kvmem_hip_pool &pool, const kvmem_hip_attn_args &a) {
    const int got = kvmem_hip_attention(&ctx, &pool, 0, &a);
    const std::string said = kvmem_hip_last_error(&ctx);
    if (got != KVMEM_HIP_ERR_INVALID || said.find("launch") == std::string::npos) {
        std::printf("%s: status %d (%s)\n", what, got, said.c_str());
        ++bad;
    }
    ctx.last_error.clear();
}

int main() {
    void *const at = reinterpret_cast<void *>(uintptr_t{0x10000});  // checked, never followed
    void *layers[1] = {at};
    kvmem_hip_pool pool{1, 8, 128, 128, 128, KVMEM_TYPE_Q4_0, KVMEM_TYPE_Q8_0, layers, layers, nullptr};
    kvmem_hip_attn_args a{};
    a.q = at, a.q_type = KVMEM_TYPE_BF16, a.out_type = KVMEM_TYPE_F32, a.q_nb1 = a.q_nb2 = 256, a.out = at;
    a.n_head = a.n_head_kv = 1, a.head_dim = 128, a.table_stride = 8, a.max_kv = 1000;
    a.q_start = a.kv_len = a.table = static_cast<uint32_t *>(at);
    // many queries: 2^21 tokens are 8192 tiles of 256 rows a request
    a.n_tokens = a.max_q = 1u << 21;
    for (uint32_t n : {1024u, 1500u, 2047u, 2048u, 65535u}) {
        a.n_seq = n;
        refused("many queries", pool, a);
    }
    // few queries: 64 rows a request are 4 tiles, times 65535 requests and 64 KV heads
    pool.n_embd_k = pool.n_embd_v = 64 * 128;
    a.n_head = a.n_head_kv = 64, a.n_seq = 65535, a.max_q = 64, a.n_tokens = 1u << 17;
    refused("few queries", pool, a);
    std::printf(bad ? "%d calls are not refused\n" : "all refused\n", bad);
    return bad ? 1 : 0;
}
